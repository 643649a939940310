// RMSNorm of every query and key head and the rotation by position, in one pass over the projections' rows.
//   y = x * rsqrt(mean(x^2) + eps) * w ;  (a, b) -> (a c - b s, a s + b c) for the pairs of dims [first, first + rot)
// Bound by memory: each value is read and written once.  Eight elements per lane, so a head of 64 / 128 / 256 dims is 8 / 16 / 32 lanes
// and a warp has 4 / 2 / 1 heads; a row's (cos, sin) factors are loaded once per lane and used for all heads of the token.
#include <algorithm>
#include "kv8.cuh"

namespace msb {

struct NormRopeParams {
  const void *q, *k;
  void *q_out, *k_out;
  const float *q_w, *k_w, *cs;
  const int* pos;
  int64_t q_stride, k_stride, q_out_stride, k_out_stride;
  int q_heads, k_heads, D, rot, first, halves, n_pos, per_block;
  int q_vec, k_vec;
  float eps;
  int* status;
};

constexpr int kNrThreads = 256;

// LANES lanes a head (a power of two >= D / 8)
template <class T, int LANES>
__global__ void __launch_bounds__(kNrThreads) head_norm_rope_kernel(const NormRopeParams p) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int kGroups = kNrThreads / LANES;
  const int lane = threadIdx.x & 31, l = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const int64_t row = blockIdx.x;
  const int pos = __ldg(p.pos + row);
  if (pos < 0) return;                                    // a padding row
  if (pos >= p.n_pos) {
    if (threadIdx.x == 0) atomicCAS(p.status, 0, kDevBadBatch);
    return;
  }
  const int d = 8 * l;
  const bool live = d < p.D, turned = live && d >= p.first && d < p.first + p.rot;
  // this lane's factors: of its four pairs, or of its eight dims' pairs (halves)
  float c[8], s[8];
  const int half = p.rot >> 1;
  const bool upper = p.halves && d - p.first >= half;     // the second member of its pairs
  if (turned) {
    const float* f = p.cs + (int64_t)pos * p.rot + (p.halves ? 2 * (d - p.first - (upper ? half : 0)) : d - p.first);
#pragma unroll
    for (int i = 0; i < 8; i++)
      if (i < 4 || p.halves) { c[i] = __ldg(f + 2 * i); s[i] = __ldg(f + 2 * i + 1); }
  }
  const int partner = lane + (upper ? -(half >> 3) : half >> 3);
  const int h0 = blockIdx.y * p.per_block, h1 = min(h0 + p.per_block, p.q_heads + p.k_heads);
  for (int hb = h0; hb < h1; hb += kGroups) {             // the same count in every warp: the shuffles below are whole
    const int h = hb + group;
    const bool mine = live && h < h1, key = h >= p.q_heads;
    const int hh = key ? h - p.q_heads : h;
    const bool vec = key ? p.k_vec : p.q_vec;
    const float* w = key ? p.k_w : p.q_w;
    float x[8], g[8];
#pragma unroll
    for (int i = 0; i < 8; i++) { x[i] = 0.f; g[i] = 1.f; }
    if (mine) {
      Elems<T>::load(static_cast<const T*>(key ? p.k : p.q) + row * (key ? p.k_stride : p.q_stride) + (int64_t)hh * p.D + d, vec, x);
      if (w) {
#pragma unroll
        for (int i = 0; i < 8; i++) g[i] = __ldg(w + d + i);
      }
    }
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) ss = fmaf(x[i], x[i], ss);
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float r = rsqrtf(ss / (float)p.D + p.eps);
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = x[i] * r * g[i];
    if (p.halves) {
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const float o = __shfl_sync(0xffffffffu, x[i], partner & 31);
        if (turned) x[i] = upper ? fmaf(o, s[i], x[i] * c[i]) : fmaf(x[i], c[i], -(o * s[i]));
      }
    } else if (turned) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float a = x[2 * i], b = x[2 * i + 1];
        x[2 * i] = fmaf(a, c[i], -(b * s[i]));
        x[2 * i + 1] = fmaf(a, s[i], b * c[i]);
      }
    }
    if (mine)
      Elems<T>::store(static_cast<T*>(key ? p.k_out : p.q_out) + row * (key ? p.k_out_stride : p.q_out_stride) + (int64_t)hh * p.D + d, vec, x);
  }
}

template <class T>
static int launch_norm_rope(NormRopeParams& p, int n_tokens, cudaStream_t st) {
  const int lanes = p.D <= 64 ? 8 : p.D <= 128 ? 16 : 32, groups = kNrThreads / lanes, heads = p.q_heads + p.k_heads;
  p.per_block = std::max(groups, n_tokens >= 1024 ? heads : groups);
  const dim3 grid((unsigned)n_tokens, (unsigned)((heads + p.per_block - 1) / p.per_block));
  auto go = [&](auto kern) { return launch_pdl(kern, grid, dim3(kNrThreads), 0, st, p); };
  MSB_CUDA(lanes == 8 ? go(head_norm_rope_kernel<T, 8>) : lanes == 16 ? go(head_norm_rope_kernel<T, 16>) : go(head_norm_rope_kernel<T, 32>));
  MSB_LAUNCH_CHECK("head_norm_rope");
  return kOk;
}

int head_norm_rope(int elem_type, const void* q, int q_heads, int64_t q_stride, const float* q_w, const void* k, int k_heads,
                   int64_t k_stride, const float* k_w, int n_tokens, int D, float eps, const float* cs, const int* pos, int n_pos, int rot,
                   int first, int halves, void* q_out, int64_t q_out_stride, void* k_out, int64_t k_out_stride, cudaStream_t st) {
  const char* what = "head_norm_rope";
  if (n_tokens <= 0 || q_heads < 0 || k_heads < 0 || q_heads + k_heads <= 0 || q_heads > 65535 || k_heads > 65535)
    return fail(kErrArg, "%s: %d rows of %d + %d heads", what, n_tokens, q_heads, k_heads);
  if (D < 8 || D > 256 || D % 8) return fail(kErrArg, "%s: head dim %d (multiples of 8 up to 256)", what, D);
  if (rot < 0 || rot % 2 || first < 0 || first + rot > D || first % 8 || rot % (halves ? 16 : 8))
    return fail(kErrArg, "%s: rotation of %d dims from %d on (first a multiple of 8, the count of 8, by halves of 16)", what, rot, first);
  if (!pos || n_pos <= 0 || (rot && !cs)) return fail(kErrArg, "%s: null pointer or no positions", what);
  NormRopeParams p{};
  bool v[4] = {true, true, true, true};
  int rc;
  if (q_heads && ((rc = kv8_rows_check(q, q_stride, q_heads, D, elem_type, what, &v[0])) ||
                  (rc = kv8_rows_check(q_out, q_out_stride, q_heads, D, elem_type, what, &v[1])))) return rc;
  if (k_heads && ((rc = kv8_rows_check(k, k_stride, k_heads, D, elem_type, what, &v[2])) ||
                  (rc = kv8_rows_check(k_out, k_out_stride, k_heads, D, elem_type, what, &v[3])))) return rc;
  Tables tb;
  if ((rc = get_tables(&tb))) return rc;
  p.q = q; p.k = k; p.q_out = q_out; p.k_out = k_out; p.q_w = q_w; p.k_w = k_w; p.cs = cs; p.pos = pos;
  p.q_stride = q_stride; p.k_stride = k_stride; p.q_out_stride = q_out_stride; p.k_out_stride = k_out_stride;
  p.q_heads = q_heads; p.k_heads = k_heads; p.D = D; p.rot = rot; p.first = first; p.halves = halves != 0; p.n_pos = n_pos;
  p.q_vec = v[0] && v[1]; p.k_vec = v[2] && v[3]; p.eps = eps; p.status = tb.status;
  return elem_type == F32 ? launch_norm_rope<float>(p, n_tokens, st) : elem_type == F16 ? launch_norm_rope<__half>(p, n_tokens, st)
                                                                                        : launch_norm_rope<__nv_bfloat16>(p, n_tokens, st);
}

}  // namespace msb
