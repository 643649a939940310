// RMSNorm of every query and key head and the rotation by position, in one pass over the projections' rows.
//   y = x * rsqrt(mean(x^2) + eps) * w ;  (a, b) -> (a c - b s, a s + b c) for the pairs of dims [first, first + rot)
// Each value is read and written once.  Eight elements per lane, so a head of 64 / 128 / 256 dims is 8 / 16 / 32 lanes and a warp has
// 4 / 2 / 1 heads at a time; the gains are multiplied into the token's (cos, sin) factors, which stay in a lane's registers for all its
// heads, and four groups of heads are on the way while four are computed: a warp's chain of loads is what bounds it (4096 tokens with 64 + 8
// heads of 128, bf16: 58 us with a block a token, 40.3 with a warp a token, 33.5 = 4.57 TB/s with the next loads ahead; neither eight groups
// nor more warps an SM with fewer registers end sooner).
#include <algorithm>
#include "kv8.cuh"

namespace msb {

struct NormRopeSide {             // the query heads, or the key heads
  const void* in;
  void* out;
  const float* w;
  int64_t in_stride, out_stride;
  int heads, vec;
};
struct NormRopeParams {
  NormRopeSide q, k;
  const float* cs;
  const int* pos;
  int n_tokens, D, rot, first, halves, n_pos, per_block, cs_vec, w_vec;
  float eps;
  int* status;
};

constexpr int kNrWarps = 4;      // tokens of a block

// LANES lanes a head (a power of two >= D / 8)
template <class T, int LANES>
__global__ void __launch_bounds__(32 * kNrWarps) head_norm_rope_kernel(const NormRopeParams p) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int kGroups = 32 / LANES;                     // heads of a warp
  typedef typename Elems<T>::Raw Raw;
  constexpr int kHeads = 4;                               // heads of a group of lanes that are under way at a time
  const int lane = threadIdx.x, l = lane % LANES, group = lane / LANES;
  const int64_t row = (int64_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (row >= p.n_tokens) return;
  const int d = 8 * l;
  const bool live = d < p.D;
  const int pos = __ldg(p.pos + row);
  if (pos < 0) return;                                    // a padding row
  if (pos >= p.n_pos) {
    if (lane == 0) atomicCAS(p.status, 0, kDevBadBatch);
    return;
  }
  const bool turned = live && d >= p.first && d < p.first + p.rot;
  const int half = p.rot >> 1;
  const bool upper = p.halves && d - p.first >= half;     // the second member of its pairs
  const int partner = turned ? lane + (upper ? -(half >> 3) : half >> 3) : lane, other = p.halves ? d + (upper ? -half : half) : d;
  const float inv_d = 1.f / (float)p.D;
  // this block's share of the query heads, then of the key heads
#pragma unroll 1
  for (int side = 0; side < 2; side++) {
    const NormRopeSide& sd = side ? p.k : p.q;
    const int from = (int)blockIdx.y * p.per_block - (side ? p.q.heads : 0), h0 = max(from, 0), h1 = min(from + p.per_block, sd.heads);
    if (h0 >= h1) continue;
    const bool vec = sd.vec;
    const float* w = sd.w;
    const T* x = static_cast<const T*>(sd.in) + row * sd.in_stride + d;
    T* y = static_cast<T*>(sd.out) + row * sd.out_stride + d;
    Raw raw[kHeads];
    auto load = [&](int hb) {
#pragma unroll
      for (int i = 0; i < kHeads; i++) {
        const int h = hb + i * kGroups;
        raw[i] = {};
        if (live && h < h1) raw[i] = vec ? Elems<T>::raw(x + h * p.D) : Elems<T>::gather(x + h * p.D);
      }
    };
    load(h0 + group);
    // with the gains in the factors: y_i = r (x_i a_i + o_i b_i), o_i the other member of the pair (of what is not turned: itself, times 0)
    float a[8], b[8];
#pragma unroll
    for (int i = 0; i < 8; i++) { a[i] = 1.f; b[i] = 0.f; }
    if (w && live) Elems<float>::load(w + d, p.w_vec, a);
    if (turned) {
      float g[8], t[8];
#pragma unroll
      for (int i = 0; i < 8; i++) g[i] = a[i];
      if (w && p.halves) Elems<float>::load(w + other, p.w_vec, g);
      const float* f = p.cs + (int64_t)pos * p.rot + (p.halves ? 2 * (d - p.first - (upper ? half : 0)) : d - p.first);
      Elems<float>::load(f, p.cs_vec, t);
      if (p.halves) {
#pragma unroll
        for (int i = 0; i < 4; i++) { a[i] *= t[2 * i]; b[i] = g[i] * (upper ? t[2 * i + 1] : -t[2 * i + 1]); }
        Elems<float>::load(f + 8, p.cs_vec, t);
#pragma unroll
        for (int i = 0; i < 4; i++) { a[4 + i] *= t[2 * i]; b[4 + i] = g[4 + i] * (upper ? t[2 * i + 1] : -t[2 * i + 1]); }
      } else {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          a[i] *= t[i]; a[i + 1] *= t[i];
          b[i] = -g[i + 1] * t[i + 1]; b[i + 1] = g[i] * t[i + 1];
        }
      }
    }
    uint64_t a2[4], b2[4];
#pragma unroll
    for (int i = 0; i < 4; i++) { a2[i] = kv8_two(a[2 * i], a[2 * i + 1]); b2[i] = kv8_two(b[2 * i], b[2 * i + 1]); }
    for (int hb = h0 + group; hb - group < h1; hb += kHeads * kGroups) {     // whole warps: the shuffles need every lane
      Raw now[kHeads];
#pragma unroll
      for (int i = 0; i < kHeads; i++) now[i] = raw[i];
      if (hb - group + kHeads * kGroups < h1) load(hb + kHeads * kGroups);   // on the way while these are computed
#pragma unroll
      for (int i = 0; i < kHeads; i++) {
        const int h = hb + i * kGroups;
        if (h - group >= h1) break;               // none of the warp's
        float v[8], o[8];
        Elems<T>::open(now[i], v);
        if (p.halves) {
          Elems<T>::open(Elems<T>::from_lane(now[i], partner), o);
        } else {
#pragma unroll
          for (int j = 0; j < 8; j++) o[j] = turned ? v[j ^ 1] : v[j];
        }
        uint64_t x2[4], ss = 0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
          x2[j] = kv8_two(v[2 * j], v[2 * j + 1]);
          ss = kv8_fma2(x2[j], x2[j], ss);
        }
        float sum, rest;
        kv8_apart(ss, sum, rest);
        sum += rest;
#pragma unroll
        for (int k = LANES / 2; k > 0; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
        const float r = rsqrtf(fmaf(sum, inv_d, p.eps));
        const uint64_t r2 = kv8_two(r, r);
#pragma unroll
        for (int j = 0; j < 4; j++)
          kv8_apart(kv8_mul2(r2, kv8_fma2(x2[j], a2[j], kv8_mul2(kv8_two(o[2 * j], o[2 * j + 1]), b2[j]))), v[2 * j], v[2 * j + 1]);
        if (live && h < h1) Elems<T>::store(y + h * p.D, vec, v);
      }
    }
  }
}

template <class T>
static int launch_norm_rope(NormRopeParams& p, int n_tokens, cudaStream_t st) {
  const int lanes = p.D <= 64 ? 8 : p.D <= 128 ? 16 : 32, groups = 32 / lanes, heads = p.q.heads + p.k.heads;
  // all heads of a token in a warp once the tokens alone fill the GPU twice; before, a head a group of lanes
  const bool many = n_tokens >= 2 * 148;
  p.per_block = many ? heads : groups;
  p.n_tokens = n_tokens;
  const int warps = many ? kNrWarps : 1;
  const dim3 grid((unsigned)((n_tokens + warps - 1) / warps), (unsigned)((heads + p.per_block - 1) / p.per_block)), block(32, warps);
  auto go = [&](auto kern) { return launch_pdl(kern, grid, block, 0, st, p); };
  MSB_CUDA(lanes == 8 ? go(head_norm_rope_kernel<T, 8>) : lanes == 16 ? go(head_norm_rope_kernel<T, 16>) : go(head_norm_rope_kernel<T, 32>));
  MSB_LAUNCH_CHECK("head_norm_rope");
  return kOk;
}

int head_norm_rope(int elem_type, const void* q, int q_heads, int64_t q_stride, const float* q_w, const void* k, int k_heads,
                   int64_t k_stride, const float* k_w, int n_tokens, int D, float eps, const float* cs, const int* pos, int n_pos, int rot,
                   int first, int halves, void* q_out, int64_t q_out_stride, void* k_out, int64_t k_out_stride, cudaStream_t st) {
  const char* what = "head_norm_rope";
  if (n_tokens <= 0 || q_heads < 0 || k_heads < 0 || q_heads + k_heads <= 0 || q_heads > 32767 || k_heads > 32767)
    return fail(kErrArg, "%s: %d rows of %d + %d heads", what, n_tokens, q_heads, k_heads);
  if (D < 8 || D > 256 || D % 8) return fail(kErrArg, "%s: head dim %d (multiples of 8 up to 256)", what, D);
  if (rot < 0 || rot % 2 || first < 0 || rot > D || first > D - rot || first % 8 || rot % (halves ? 16 : 8))
    return fail(kErrArg, "%s: rotation of %d dims from %d on (first a multiple of 8, the count of 8, by halves of 16)", what, rot, first);
  if (!pos || n_pos <= 0 || (rot && !cs)) return fail(kErrArg, "%s: null pointer or no positions", what);
  if ((reinterpret_cast<uintptr_t>(pos) | reinterpret_cast<uintptr_t>(cs) | reinterpret_cast<uintptr_t>(q_w) | reinterpret_cast<uintptr_t>(k_w)) & 3)
    return fail(kErrArg, "%s: positions, factors or gains are not aligned to their elements", what);
  NormRopeParams p{};
  bool v[4] = {true, true, true, true};
  int rc;
  if (q_heads && ((rc = kv8_rows_check(q, q_stride, q_heads, D, elem_type, what, &v[0])) ||
                  (rc = kv8_rows_check(q_out, q_out_stride, q_heads, D, elem_type, what, &v[1])))) return rc;
  if (k_heads && ((rc = kv8_rows_check(k, k_stride, k_heads, D, elem_type, what, &v[2])) ||
                  (rc = kv8_rows_check(k_out, k_out_stride, k_heads, D, elem_type, what, &v[3])))) return rc;
  Tables tb;
  if ((rc = get_tables(&tb))) return rc;
  p.q = NormRopeSide{q, q_out, q_w, q_stride, q_out_stride, q_heads, v[0] && v[1]};
  p.k = NormRopeSide{k, k_out, k_w, k_stride, k_out_stride, k_heads, v[2] && v[3]};
  p.cs = cs; p.pos = pos; p.D = D; p.rot = rot; p.first = first; p.halves = halves != 0; p.n_pos = n_pos;
  p.cs_vec = reinterpret_cast<uintptr_t>(cs) % 16 == 0 && rot % 4 == 0;
  p.w_vec = (reinterpret_cast<uintptr_t>(q_w) | reinterpret_cast<uintptr_t>(k_w)) % 16 == 0;
  p.eps = eps; p.status = tb.status;
  return elem_type == F32 ? launch_norm_rope<float>(p, n_tokens, st) : elem_type == F16 ? launch_norm_rope<__half>(p, n_tokens, st)
                                                                                        : launch_norm_rope<__nv_bfloat16>(p, n_tokens, st);
}

}  // namespace msb
