// Writing new key / value rows into the 8-bit cache (kv8.cuh) and reading rows back.
//   scale = 2^E, E the smallest of [-50, 50] with max |x| <= 448 * 2^E over the block's values of one head (50 where there is none);
//   code = e4m3(x / scale), nearest even, +-448 beyond
// When a block already holds older tokens its scale only grows: E = max(E of the new values, E so far), and the older codes are
// rounded to e4m3 again after division by the power of two (exact but for what falls below the format's normal range, 2^-6).
// Both kernels move each byte once and are bound by memory, or for few tokens by the chain of look-ups: the sequence of a work item,
// its lengths, its block.  A group of threads does that once and goes over several (head, keys or values) units of the block: it holds a
// unit's new values in registers between the maximum and the rounding, and the next unit's are on the way meanwhile.
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
  if ((reinterpret_cast<uintptr_t>(c->k_scale) | reinterpret_cast<uintptr_t>(c->v_scale)) & 3) return fail(kErrArg, "%s: scales are not aligned to F32", what);
  if (b->n_seq <= 0 || b->n_seq > 65535) return fail(kErrArg, "%s: %d sequences (1 to 65535)", what, b->n_seq);
  if (b->n_tokens <= 0 || b->max_new <= 0 || b->max_new > b->n_tokens) return fail(kErrArg, "%s: %d rows, at most %d new ones", what, b->n_tokens, b->max_new);
  if (b->max_len < b->max_new || b->max_len > (1 << 30)) return fail(kErrArg, "%s: at most %d tokens, %d of them new", what, b->max_len, b->max_new);
  if (b->table_stride <= 0 || (int64_t)b->table_stride * c->block < b->max_len)
    return fail(kErrArg, "%s: %d blocks of %d tokens do not hold %d", what, b->table_stride, c->block, b->max_len);
  if (!b->seq_start || !b->kv_len || !b->table) return fail(kErrArg, "%s: null pointer in the batch", what);
  if ((reinterpret_cast<uintptr_t>(b->seq_start) | reinterpret_cast<uintptr_t>(b->kv_len) | reinterpret_cast<uintptr_t>(b->table)) & 3)
    return fail(kErrArg, "%s: the batch's arrays are not aligned to int32", what);
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
  int each;                       // items of a sequence, 0: as Kv8Items finds them
  int* status;
};

constexpr int kKv8Threads = 256;
constexpr int kv8_block_threads(int group) { return group > kKv8Threads ? group : kKv8Threads; }

// THREADS threads a unit (whole warps), each with up to MOST pieces of eight values
template <class T, int D, int THREADS, int MOST>
__global__ void __launch_bounds__(kv8_block_threads(THREADS)) kv8_write_kernel(const Kv8RowsParams p) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int kGroups = kv8_block_threads(THREADS) / THREADS, kRow = D / 8, kWarps = THREADS / 32;
  __shared__ float s_top[kGroups][2][kWarps];
  float (&s_max)[2][kWarps] = s_top[threadIdx.x / THREADS];
  const int tid = threadIdx.x % THREADS, sh = p.c.shift, units = 2 * p.c.heads, step = gridDim.y * kGroups;
  Kv8Items items;
  Kv8Item it;
  for (int s, turn = 0; items.next(p.b, sh, p.each, blockIdx.x, p.status, s, it);) {
    const int pieces = it.n * kRow;
    typename Elems<T>::Raw r[MOST], next[MOST];
    auto load = [&](int u) {        // unit u: head u / 2, its keys or its values
      const bool values = u & 1, vec = values ? p.v_vec : p.k_vec;
      const int64_t stride = values ? p.v_stride : p.k_stride;
      const T* rows = static_cast<const T*>(values ? p.v : p.k) + it.row * stride + (u >> 1) * D;
      if (vec) {
#pragma unroll
        for (int i = 0; i < MOST; i++) {
          const int c = tid + i * THREADS;
          if (c < pieces) next[i] = Elems<T>::raw(rows + (c / kRow) * stride + c % kRow * 8);
        }
      } else {
#pragma unroll
        for (int i = 0; i < MOST; i++) {
          const int c = tid + i * THREADS;
          if (c < pieces) next[i] = Elems<T>::gather(rows + (c / kRow) * stride + c % kRow * 8);
        }
      }
    };
    int u = blockIdx.y * kGroups + threadIdx.x / THREADS;
    if (u < units) load(u);
    const int id = kv8_block(p.b, p.c.n_blocks, s, it, p.status);
    if (id < 0) continue;
    float was = 0.f;
    if (it.at && u < units) was = ((u & 1) ? p.c.vs : p.c.ks)[(size_t)id * p.c.heads + (u >> 1)];
    for (; u < units; u += step, turn ^= 1) {
      const size_t head = (size_t)id * p.c.heads + (u >> 1);
      uint8_t* codes = ((u & 1) ? p.c.v : p.c.k) + (head << sh) * D;
      float* scale = ((u & 1) ? p.c.vs : p.c.ks) + head;
      const float old = was;
#pragma unroll
      for (int i = 0; i < MOST; i++) r[i] = next[i];
      if (u + step < units) {
        load(u + step);
        if (it.at) was = (((u + step) & 1) ? p.c.vs : p.c.ks)[(size_t)id * p.c.heads + ((u + step) >> 1)];
      }
      float top = 0.f;
      bool nan = false;
#pragma unroll
      for (int i = 0; i < MOST; i++)
        if (tid + i * THREADS < pieces) {
          float v[8];
          Elems<T>::open(r[i], v);
#pragma unroll
          for (int j = 0; j < 8; j++) {
            const float a = fabsf(v[j]);
            nan |= a != a;
            if (a <= 3.402823466e38f) top = fmaxf(top, a);            // an infinity becomes the largest code
          }
        }
      top = warp_max(top);
      if (THREADS > 32) {
        if ((tid & 31) == 0) s_max[turn][tid >> 5] = top;
        bar_sync_named(1 + threadIdx.x / THREADS, THREADS);           // (also: every thread has read the scale that is written below)
#pragma unroll
        for (int i = 0; i < kWarps; i++) top = fmaxf(top, s_max[turn][i]);
      }
      // top = 1.m * 2^e <= 448 * 2^E = 1.75 * 2^(8 + E)
      const uint32_t bits = __float_as_uint(top);
      int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
      e = min(max(e, kKv8MinExp), kKv8MaxExp);
      int e_old = e;
      if (it.at) { e_old = kv8_exp(old); e = max(e, e_old); }
      const float inv = kv8_pow2(-e);
#pragma unroll
      for (int i = 0; i < MOST; i++) {
        const int c = tid + i * THREADS;
        if (c < pieces) {
          float v[8];
          Elems<T>::open(r[i], v);
#pragma unroll
          for (int j = 0; j < 8; j++) v[j] *= inv;
          if (nan) {                                                  // the cache holds none: its attention multiplies masked rows by 0
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = v[j] != v[j] ? 0.f : v[j];
          }
          *reinterpret_cast<uint2*>(codes + (it.at + c / kRow) * D + c % kRow * 8) =
              make_uint2(kv8_codes4(v[0], v[1], v[2], v[3]), kv8_codes4(v[4], v[5], v[6], v[7]));
        }
      }
      if (nan) atomicCAS(p.status, 0, kDevNan);
      if (e > e_old) {                                                // older tokens of the block move to the larger scale
        const float f = kv8_pow2(e_old - e);
#pragma unroll 4
        for (int c = tid; c < it.at * (D / 16); c += THREADS) {
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
      if (THREADS == 32) __syncwarp();
      if (tid == 0) *scale = kv8_pow2(e);
    }
  }
}

// 16 bytes of a row a thread and step: eight values, four of F32; THREADS threads a unit, up to MOST steps
template <class T, int D, int THREADS, int MOST>
__global__ void __launch_bounds__(kKv8Threads) kv8_read_kernel(const Kv8RowsParams p) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int V = 16 / sizeof(T), kRow = D / V, kGroups = kKv8Threads / THREADS;
  const int sh = p.c.shift, units = 2 * p.c.heads, tid = threadIdx.x % THREADS, step = gridDim.y * kGroups;
  Kv8Items items;
  Kv8Item it;
  for (int s; items.next(p.b, sh, p.each, blockIdx.x, p.status, s, it);) {
    const int id = kv8_block(p.b, p.c.n_blocks, s, it, p.status), pieces = it.n * kRow;
    uint32_t w[MOST][V / 4], next[MOST][V / 4] = {};
    float scale = 0.f, next_scale = 0.f;
    auto load = [&](int u) {
      if (id < 0) return;
      const size_t head = (size_t)id * p.c.heads + (u >> 1);
      const uint8_t* codes = ((u & 1) ? p.c.v : p.c.k) + (head << sh) * D + it.at * D;
#pragma unroll
      for (int i = 0; i < MOST; i++) {
        const int c = tid + i * THREADS;
        if (c < pieces) {
          if (V == 8) {
            const uint2 q = __ldg(reinterpret_cast<const uint2*>(codes) + c);
            next[i][0] = q.x; next[i][V / 4 - 1] = q.y;
          } else {
            next[i][0] = __ldg(reinterpret_cast<const uint32_t*>(codes) + c);
          }
        }
      }
      next_scale = __ldg(((u & 1) ? p.c.vs : p.c.ks) + head);
    };
    int u = blockIdx.y * kGroups + threadIdx.x / THREADS;
    if (u < units) load(u);
    for (; u < units; u += step) {
#pragma unroll
      for (int i = 0; i < MOST; i++)
#pragma unroll
        for (int j = 0; j < V / 4; j++) w[i][j] = next[i][j];
      scale = next_scale;
      if (u + step < units) load(u + step);
      const bool values = u & 1, vec = values ? p.v_vec : p.k_vec;
      const int64_t stride = values ? p.v_stride : p.k_stride;
      T* rows = static_cast<T*>(values ? p.v : p.k) + it.row * stride + (u >> 1) * D;
#pragma unroll
      for (int i = 0; i < MOST; i++) {
        const int c = tid + i * THREADS;
        if (c >= pieces) break;
        float o[V];
#pragma unroll
        for (int j = 0; j < V / 2; j++) {
          const float2 a = kv8_float2(w[i][j >> 1] >> (16 * (j & 1)));
          o[2 * j] = a.x * scale; o[2 * j + 1] = a.y * scale;
        }
        Elems<T>::store16(rows + (c / kRow) * stride + c % kRow * V, vec, o);
      }
    }
  }
}

template <class T, int D>
static int launch_rows(bool write, Kv8RowsParams& p, cudaStream_t st) {
  const int sh = p.c.shift, units = 2 * p.c.heads;
  // items: every sequence's most, or as its rows have it
  const int64_t each = kv8_touched(p.b.max_new, sh), all = kv8_items(p.b.n_tokens, p.b.n_seq, sh);
  p.each = each * p.b.n_seq <= all ? (int)each : 0;
  const int64_t items = p.each ? each * p.b.n_seq : all + 1;             // (and one more that looks for what the search misses)
  if (items > 0x7fffffff) return fail(kErrLimit, "kv8: too many rows");
  // blocks of threads of `group` threads a unit, each over `per` units while there are blocks enough for every SM
  auto go = [&](auto kern, int group, int64_t an_sm) {
    const int groups = kv8_block_threads(group) / group, per = (int)std::max<int64_t>(1, std::min<int64_t>(units, items * units / (148 * an_sm * groups)));
    return launch_pdl(kern, dim3((unsigned)items, (units + per * groups - 1) / (per * groups)), dim3(kv8_block_threads(group)), 0, st, p);
  };
  const int pieces = (D / 8) << sh;
  if (!write) {
    // (16 sequences of up to 8192 tokens, blocks of 64: 90.5 us with 4 or 8 blocks an SM, 84.7 with 16, 82.6 with 32, 87.3 with 64; blocks of
    // 16 tokens with 256 threads for all: 124)
    const int steps = (D * (int)sizeof(T) / 16) << sh;
    MSB_CUDA(steps <= 128 ? go(kv8_read_kernel<T, D, 32, 4>, 32, 32) : steps <= 256 ? go(kv8_read_kernel<T, D, 64, 4>, 64, 32)
             : steps <= 512 ? go(kv8_read_kernel<T, D, 128, 4>, 128, 32) : steps <= 1024 ? go(kv8_read_kernel<T, D, 256, 4>, 256, 32)
             : steps <= 2048 ? go(kv8_read_kernel<T, D, 256, 8>, 256, 32) : go(kv8_read_kernel<T, D, 256, 16>, 256, 32));
  } else if ((int64_t)std::min(p.b.max_new, 1 << sh) * (D / 8) <= 64) {
    MSB_CUDA(go(kv8_write_kernel<T, D, 32, 2>, 32, 1 << 20));       // few new rows: a warp a unit
  } else {
    // four pieces a thread, whatever the block (ragged prompts, bf16, blocks of 16 / 64 / 128 tokens: 19.7 / 17.8 / 23.5 us; with 256 threads
    // for all of them 31.3 / 17.3 / 31.2)
    MSB_CUDA(pieces <= 128 ? go(kv8_write_kernel<T, D, 32, 4>, 32, 4) : pieces <= 256 ? go(kv8_write_kernel<T, D, 64, 4>, 64, 4)
             : pieces <= 512 ? go(kv8_write_kernel<T, D, 128, 4>, 128, 4) : pieces <= 1024 ? go(kv8_write_kernel<T, D, 256, 4>, 256, 4)
                                                                                   : go(kv8_write_kernel<T, D, 512, 4>, 512, 4));
  }
  MSB_LAUNCH_CHECK(write ? "kv8_write" : "kv8_read");
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
#define KV8_GO(T) return c->head_dim == 64 ? launch_rows<T, 64>(write, p, st) : launch_rows<T, 128>(write, p, st)
  if (elem_type == F32) KV8_GO(float);
  if (elem_type == F16) KV8_GO(__half);
  KV8_GO(__nv_bfloat16);
#undef KV8_GO
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
