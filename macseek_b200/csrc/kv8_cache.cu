// Writing new key / value rows into the 8-bit cache (kv8.cuh) and reading rows back.
//   scale = 2^E, E the smallest of [-50, 50] with max |x| <= 448 * 2^E over the block's values of one head (50 where there is none);
//   code = e4m3(x / scale), nearest even, +-448 beyond
// When a block already holds older tokens its scale only grows: E = max(E of the new values, E so far), and the older codes are
// rounded to e4m3 again after division by the power of two (exact but for what falls below the format's normal range, 2^-6).
// Both kernels move each byte once and are bound by memory: one block of threads per (cache block, head, keys or values), which holds
// all its new values in registers between the maximum and the rounding.
#include <algorithm>
#include "kv8.cuh"

namespace msb {

int kv8_check(const msb_kv8_cache* c, const msb_kv8_batch* b, const char* what, Kv8Cache* cc, Kv8Batch* bb) {
  if (!c || !b) return fail(kErrArg, "%s: null cache or batch", what);
  if (c->n_blocks <= 0 || c->kv_heads <= 0 || c->kv_heads > 1024) return fail(kErrArg, "%s: %d blocks of %d heads", what, c->n_blocks, c->kv_heads);
  if (c->head_dim != 64 && c->head_dim != 128) return fail(kErrArg, "%s: head dim %d is not 64 or 128", what, c->head_dim);
  if (c->block != 16 && c->block != 32 && c->block != 64 && c->block != 128)
    return fail(kErrArg, "%s: %d tokens in a block (16, 32, 64 or 128)", what, c->block);
  if (!c->k || !c->v || !c->k_scale || !c->v_scale) return fail(kErrArg, "%s: null pointer in the cache", what);
  if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15) return fail(kErrArg, "%s: codes must be 16-byte aligned", what);
  if (b->n_seq <= 0 || b->n_seq > 65535) return fail(kErrArg, "%s: %d sequences (1 to 65535)", what, b->n_seq);
  if (b->n_tokens <= 0 || b->max_new <= 0 || b->max_new > b->n_tokens) return fail(kErrArg, "%s: %d rows, at most %d new ones", what, b->n_tokens, b->max_new);
  if (b->max_len < b->max_new || b->max_len > (1 << 30)) return fail(kErrArg, "%s: at most %d tokens, %d of them new", what, b->max_len, b->max_new);
  if (b->table_stride <= 0 || (int64_t)b->table_stride * c->block < b->max_len)
    return fail(kErrArg, "%s: %d blocks of %d tokens do not hold %d", what, b->table_stride, c->block, b->max_len);
  if (!b->seq_start || !b->kv_len || !b->table) return fail(kErrArg, "%s: null pointer in the batch", what);
  int shift = 4;
  while ((1 << shift) < c->block) shift++;
  *cc = Kv8Cache{(uint8_t*)c->k, (uint8_t*)c->v, c->k_scale, c->v_scale, c->n_blocks, c->kv_heads, shift};
  *bb = Kv8Batch{b->seq_start, b->kv_len, b->table, b->n_seq, b->n_tokens, b->max_new, b->max_len, b->table_stride};
  return kOk;
}

int kv8_rows_check(const void* p, int64_t stride, int heads, int dim, int elem_type, const char* what, bool* vec) {
  if (!p) return fail(kErrArg, "%s: null pointer", what);
  if (elem_type != F32 && elem_type != F16 && elem_type != BF16) return fail(kErrType, "%s: rows must be F32, F16 or BF16", what);
  if (stride < (int64_t)heads * dim) return fail(kErrArg, "%s: stride %lld below %d heads of %d", what, (long long)stride, heads, dim);
  const int size = elem_type == F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(p) % size) return fail(kErrArg, "%s: rows are not aligned to their elements", what);
  *vec = reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * size % 16 == 0;
  return kOk;
}

struct Kv8RowsParams {
  Kv8Cache c;
  Kv8Batch b;
  void *k, *v;                    // rows (read by the writing kernel, written by the reading one)
  int64_t k_stride, v_stride;     // elements
  int k_vec, v_vec;
  int* status;
};

constexpr int kKv8Threads = 256, kKv8Most = 128 * 128 / 8 / kKv8Threads;     // pieces of eight values a thread holds at most

template <class T, int D>
__global__ void __launch_bounds__(kKv8Threads) kv8_write_kernel(const Kv8RowsParams p) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ float s_max[kKv8Threads / 32];
  const int tid = threadIdx.x, h = blockIdx.y, sh = p.c.shift;
  const bool values = blockIdx.z;
  int id;
  const Kv8Item it = kv8_item(p.b, p.c, blockIdx.x, p.status, id);
  if (it.n == 0 || id < 0) return;
  const size_t head = (size_t)id * p.c.heads + h;
  uint8_t* codes = (values ? p.c.v : p.c.k) + ((head << sh) * D);
  float* scale = (values ? p.c.vs : p.c.ks) + head;
  const int64_t stride = values ? p.v_stride : p.k_stride;
  const bool vec = values ? p.v_vec : p.k_vec;
  const T* rows = static_cast<const T*>(values ? p.v : p.k) + it.row * stride + (int64_t)h * D;
  const float was = it.at ? *scale : 0.f;
  const int pieces = it.n * (D / 8);

  float v[kKv8Most][8];
  float top = 0.f;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < kKv8Most; i++) {
    const int c = tid + i * kKv8Threads;
    if (c < pieces) Elems<T>::load(rows + (c / (D / 8)) * stride + c % (D / 8) * 8, vec, v[i]);
  }
#pragma unroll
  for (int i = 0; i < kKv8Most; i++) {
    if (tid + i * kKv8Threads < pieces)
#pragma unroll
      for (int j = 0; j < 8; j++) {
        if (v[i][j] != v[i][j]) { nan = true; v[i][j] = 0.f; }      // the cache holds no NaN: its attention multiplies masked rows by 0
        const float a = fabsf(v[i][j]);
        if (a <= 3.402823466e38f) top = fmaxf(top, a);              // an infinity becomes the largest code
      }
  }
  if (nan) atomicCAS(p.status, 0, kDevNan);
  top = warp_max(top);
  if ((tid & 31) == 0) s_max[tid >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kKv8Threads / 32; i++) top = fmaxf(top, s_max[i]);
  // top = 1.m * 2^e <= 448 * 2^E = 1.75 * 2^(8 + E)
  const uint32_t u = __float_as_uint(top);
  int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  e = min(max(e, kKv8MinExp), kKv8MaxExp);
  int e_old = e;
  if (it.at) { e_old = kv8_exp(was); e = max(e, e_old); }
  const float inv = kv8_pow2(-e);
#pragma unroll
  for (int i = 0; i < kKv8Most; i++) {
    const int c = tid + i * kKv8Threads;
    if (c < pieces)
      *reinterpret_cast<uint2*>(codes + (it.at + c / (D / 8)) * D + c % (D / 8) * 8) =
          make_uint2(kv8_codes4(v[i][0] * inv, v[i][1] * inv, v[i][2] * inv, v[i][3] * inv),
                     kv8_codes4(v[i][4] * inv, v[i][5] * inv, v[i][6] * inv, v[i][7] * inv));
  }
  if (e > e_old) {                                                  // older tokens of the block move to the larger scale
    const float f = kv8_pow2(e_old - e);
    for (int c = tid; c < it.at * (D / 16); c += kKv8Threads) {
      uint4* q = reinterpret_cast<uint4*>(codes) + c;
      uint32_t w[4] = {q->x, q->y, q->z, q->w};
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float2 a = kv8_float2(w[j]), b = kv8_float2(w[j] >> 16);
        w[j] = kv8_codes4(a.x * f, a.y * f, b.x * f, b.y * f);
      }
      *q = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  if (tid == 0) *scale = kv8_pow2(e);                               // every thread read it before the barrier above
}

template <class T, int D>
__global__ void __launch_bounds__(kKv8Threads) kv8_read_kernel(const Kv8RowsParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int h = blockIdx.y, sh = p.c.shift;
  const bool values = blockIdx.z;
  int id;
  const Kv8Item it = kv8_item(p.b, p.c, blockIdx.x, p.status, id);
  if (it.n == 0) return;
  const size_t head = (size_t)max(id, 0) * p.c.heads + h;
  const uint8_t* codes = (values ? p.c.v : p.c.k) + (head << sh) * D + it.at * D;
  const float scale = id < 0 ? 0.f : (values ? p.c.vs : p.c.ks)[head];
  const int64_t stride = values ? p.v_stride : p.k_stride;
  const bool vec = values ? p.v_vec : p.k_vec;
  T* rows = static_cast<T*>(values ? p.v : p.k) + it.row * stride + (int64_t)h * D;
  for (int c = threadIdx.x; c < it.n * (D / 16); c += kKv8Threads) {
    uint4 q = make_uint4(0, 0, 0, 0);
    if (id >= 0) q = reinterpret_cast<const uint4*>(codes)[c];
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
    T* dst = rows + (c / (D / 16)) * stride + c % (D / 16) * 16;
#pragma unroll
    for (int half = 0; half < 2; half++) {
      float o[8];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const float2 a = kv8_float2(w[2 * half + (j >> 1)] >> (16 * (j & 1)));
        o[2 * j] = a.x * scale; o[2 * j + 1] = a.y * scale;
      }
      Elems<T>::store(dst + 8 * half, vec, o);
    }
  }
}

template <bool WRITE, class T>
static int launch_rows(const Kv8RowsParams& p, int D, cudaStream_t st) {
  const dim3 grid((unsigned)kv8_items(p.b.n_tokens, p.b.n_seq, p.c.shift), p.c.heads, 2);
  auto go = [&](auto kern) { return launch_pdl(kern, grid, dim3(kKv8Threads), 0, st, p); };
  if (WRITE) MSB_CUDA(D == 64 ? go(kv8_write_kernel<T, 64>) : go(kv8_write_kernel<T, 128>));
  else MSB_CUDA(D == 64 ? go(kv8_read_kernel<T, 64>) : go(kv8_read_kernel<T, 128>));
  MSB_LAUNCH_CHECK(WRITE ? "kv8_write" : "kv8_read");
  return kOk;
}

static int kv8_rows(bool write, const msb_kv8_cache* c, const msb_kv8_batch* b, int elem_type, void* k, void* v, int64_t k_stride,
                    int64_t v_stride, cudaStream_t st) {
  const char* what = write ? "kv8_write" : "kv8_read";
  Kv8RowsParams p{};
  int rc = kv8_check(c, b, what, &p.c, &p.b);
  if (rc) return rc;
  bool kvec, vvec;
  if ((rc = kv8_rows_check(k, k_stride, c->kv_heads, c->head_dim, elem_type, what, &kvec))) return rc;
  if ((rc = kv8_rows_check(v, v_stride, c->kv_heads, c->head_dim, elem_type, what, &vvec))) return rc;
  Tables tb;
  if ((rc = get_tables(&tb))) return rc;
  p.k = k; p.v = v; p.k_stride = k_stride; p.v_stride = v_stride; p.k_vec = kvec; p.v_vec = vvec; p.status = tb.status;
  const int D = c->head_dim;
  if (write)
    return elem_type == F32 ? launch_rows<true, float>(p, D, st) : elem_type == F16 ? launch_rows<true, __half>(p, D, st)
                                                                                    : launch_rows<true, __nv_bfloat16>(p, D, st);
  return elem_type == F32 ? launch_rows<false, float>(p, D, st) : elem_type == F16 ? launch_rows<false, __half>(p, D, st)
                                                                                   : launch_rows<false, __nv_bfloat16>(p, D, st);
}
int kv8_write(const msb_kv8_cache* c, const msb_kv8_batch* b, int elem_type, const void* k, const void* v, int64_t k_stride,
              int64_t v_stride, cudaStream_t st) {
  return kv8_rows(true, c, b, elem_type, const_cast<void*>(k), const_cast<void*>(v), k_stride, v_stride, st);
}
int kv8_read(const msb_kv8_cache* c, const msb_kv8_batch* b, int elem_type, void* k, void* v, int64_t k_stride, int64_t v_stride,
             cudaStream_t st) {
  return kv8_rows(false, c, b, elem_type, k, v, k_stride, v_stride, st);
}

}  // namespace msb
