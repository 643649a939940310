// The 8-bit key / value cache of grouped-query heads: what its kernels share.
//   codes   [n_blocks][kv_heads][block][dim] e4m3 bytes, keys and values apart; a block holds `block` tokens of one sequence
//   scales  [n_blocks][kv_heads] f32 powers of two, keys and values apart: value = code * scale
//   batch   seq_start [n_seq + 1]: rows of a call's new tokens; kv_len [n_seq]: tokens of the sequence, the new ones last;
//           table [n_seq][table_stride]: the sequence's blocks in order
// Powers of two: a code moves from one scale to a larger one by its exponent alone, so a block whose largest value grows token by
// token keeps its older codes' mantissas, and values and codes convert without a rounding of the scale.
#pragma once
#include <type_traits>
#include "msb_common.cuh"
#include "kv8_index.h"
#include "../../include/macseek_b200.h"

namespace msb {

enum : int { kDevBadBatch = 4, kDevNan = 5 };    // more codes of the device failure word
// Exponents of scales.  The attention's weights carry the value scales, so that a sum of weights spans their range as well: with 100 binades
// a token whose weight falls below 32 bits' range is 2^-26 of the sum at most.  (The products take weights as halves, which lose what lies 2^-32
// (F32 rows of many, 2^-43; few rows 2^-36) below the row's largest, code for code.)
constexpr int kKv8MinExp = -50, kKv8MaxExp = 50;

struct Kv8Cache {
  uint8_t *k, *v;
  float *ks, *vs;
  int n_blocks, heads, shift;      // block = 1 << shift tokens
};
struct Kv8Batch {
  const int *seq_start, *kv_len, *table;
  int n_seq, n_tokens, max_new, max_len, table_stride;
};
// checks of the two structures on the host; fills the kernels' forms
int kv8_check(const msb_kv8_cache* c, const msb_kv8_batch* b, const char* what, Kv8Cache* cc, Kv8Batch* bb);
// A row of `dim` elements for each of `heads` heads at p + row * stride: pointer and stride, and whether 16-byte accesses are aligned.
int kv8_rows_check(const void* p, int64_t stride, int heads, int dim, int elem_type, const char* what, bool* vec);

#ifdef __CUDACC__
// Sequence s of the batch, or an empty one where its numbers cannot be right (recorded).
__device__ __forceinline__ Kv8Seq kv8_seq(const Kv8Batch& b, int s, int* status) {
  Kv8Seq q;
  if (!kv8_seq_of(__ldg(b.seq_start + s), __ldg(b.seq_start + s + 1), __ldg(b.kv_len + s), b.n_tokens, b.max_new, b.max_len, q))
    atomicCAS(status, 0, kDevBadBatch);
  return q;
}
// The items of a block of threads, by whole warps.  `each` > 0: item `item` is sequence item / each's.  0: item - 1 is found among the sequences'
// first items, and the block of item 0 looks the batch through: what the others miss, which takes starts that fall, it does itself.
struct Kv8Items {
  int s = 0, j = 0;               // item 0: where the batch has been looked through to; j -1: the only item is done
  __device__ __forceinline__ bool next(const Kv8Batch& b, int shift, int each, int item, int* status, int& seq, Kv8Item& it) {
    const auto ballot = [](auto f) { return __ballot_sync(0xffffffffu, f(threadIdx.x & 31)); };
    const auto start = [&](int i) { return __ldg(b.seq_start + i); };
    if (each || item) {
      if (j < 0) return false;
      j = -1;
      if (each) {
        seq = item / each;
        it = kv8_item_of(kv8_seq(b, seq, status), item - seq * each, shift);
      } else {
        const auto first = [&](int i) { return kv8_first_item(start(i), i, shift); };
        seq = kv8_search(b.n_seq, item - 1, first, ballot);
        it = kv8_item_of(kv8_seq(b, seq, status), item - 1 - first(seq), shift);
      }
      return it.n != 0;
    }
    if (s == 0 && j == 0) {
      bool falls = false;
      for (int i = threadIdx.x & 31; i < b.n_seq; i += 32) {
        falls |= start(i + 1) < start(i);
        kv8_seq(b, i, status);                                          // (recorded, whether or not an item is found to be its)
      }
      if (!__any_sync(0xffffffffu, falls)) return false;
    }
    const bool more = kv8_next_missed(b.n_seq, shift, [&](int i) { return kv8_seq(b, i, status); }, start, ballot, s, j, it);
    seq = s;
    return more;
  }
};
// The block of an item of sequence s (-1: not there).
__device__ __forceinline__ int kv8_block(const Kv8Batch& b, int n_blocks, int s, const Kv8Item& it, int* status) {
  const int id = __ldg(b.table + (size_t)s * b.table_stride + it.blk);
  if (id >= 0 && id < n_blocks) return id;
  atomicCAS(status, 0, kDevBadBatch);
  return -1;
}

// two f32 at a time
__device__ __forceinline__ uint64_t kv8_two(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void kv8_apart(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t kv8_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t kv8_add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t kv8_mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float kv8_pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }    // -126 <= e <= 127
__device__ __forceinline__ int kv8_exp(float scale) {
  return min(max((int)(__float_as_uint(scale) >> 23 & 0xFF) - 127, kKv8MinExp), kKv8MaxExp);
}
// two codes -> two halves (exact)
__device__ __forceinline__ uint32_t kv8_half2(uint32_t codes) {
  uint32_t r;
  asm("{\n\t.reg .b16 c;\n\tcvt.u16.u32 c, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, c;\n\t}" : "=r"(r) : "r"(codes));
  return r;
}
__device__ __forceinline__ float2 kv8_float2(uint32_t codes) {
  const uint32_t h = kv8_half2(codes);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
// four values -> four codes, nearest even, beyond the format: its largest value
__device__ __forceinline__ uint32_t kv8_codes4(float a, float b, float c, float d) {
  uint32_t r;
  asm("{\n\t.reg .b16 l, h;\n\tcvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n\tmov.b32 %0, {l, h};\n\t}"
      : "=r"(r) : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}

template <class T>
__device__ __forceinline__ uint32_t kv8_pack2(float a, float b) {
  if (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint4 kv8_from_lane(const uint4& v, int lane) {
  return make_uint4(__shfl_sync(0xffffffffu, v.x, lane), __shfl_sync(0xffffffffu, v.y, lane), __shfl_sync(0xffffffffu, v.z, lane),
                    __shfl_sync(0xffffffffu, v.w, lane));
}
// eight elements of a row; vec: 16-byte aligned (raw: always)
template <class T> struct Elems;
template <> struct Elems<float> {
  struct Raw { uint4 a, b; };                                         // eight elements as they lie in memory
  static __device__ __forceinline__ Raw raw(const float* p) { return Raw{reinterpret_cast<const uint4*>(p)[0], reinterpret_cast<const uint4*>(p)[1]}; }
  static __device__ __forceinline__ Raw from_lane(const Raw& r, int lane) { return Raw{kv8_from_lane(r.a, lane), kv8_from_lane(r.b, lane)}; }
  static __device__ __forceinline__ Raw gather(const float* p) {       // not aligned
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; i++) w[i] = __float_as_uint(p[i]);
    return Raw{make_uint4(w[0], w[1], w[2], w[3]), make_uint4(w[4], w[5], w[6], w[7])};
  }
  static __device__ __forceinline__ uint4 pack16(const float (&v)[8], int k) {     // 16 bytes of eight elements' 32
    return make_uint4(__float_as_uint(v[4 * k]), __float_as_uint(v[4 * k + 1]), __float_as_uint(v[4 * k + 2]), __float_as_uint(v[4 * k + 3]));
  }
  static __device__ __forceinline__ void store16(float* p, bool vec, const float (&v)[4]) {
    if (vec) {
      *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) p[i] = v[i];
    }
  }
  static __device__ __forceinline__ void open(const Raw& r, float (&v)[8]) {
    const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = __uint_as_float(w[i]);
  }
  static __device__ __forceinline__ void load(const float* p, bool vec, float (&v)[8]) {
    if (vec) {
      open(raw(p), v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = p[i];
    }
  }
  static __device__ __forceinline__ void store(float* p, bool vec, const float (&v)[8]) {
    if (vec) {
      reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) p[i] = v[i];
    }
  }
  static __device__ __forceinline__ float from(float x) { return x; }
};
template <class T, class T2> struct Elems16 {
  typedef uint4 Raw;
  static __device__ __forceinline__ Raw raw(const T* p) { return *reinterpret_cast<const uint4*>(p); }
  static __device__ __forceinline__ Raw from_lane(const Raw& r, int lane) { return kv8_from_lane(r, lane); }
  static __device__ __forceinline__ Raw gather(const T* p) {           // not aligned
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      T2 h;
      h.x = p[2 * i]; h.y = p[2 * i + 1];
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  static __device__ __forceinline__ uint4 pack16(const float (&v)[8], int) {
    return make_uint4(kv8_pack2<T>(v[0], v[1]), kv8_pack2<T>(v[2], v[3]), kv8_pack2<T>(v[4], v[5]), kv8_pack2<T>(v[6], v[7]));
  }
  static __device__ __forceinline__ void store16(T* p, bool vec, const float (&v)[8]) { Elems16::store(p, vec, v); }
  static __device__ __forceinline__ void open(const Raw& u, float (&v)[8]) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const T2 h = *reinterpret_cast<const T2*>(&w[i]);
      v[2 * i] = static_cast<float>(h.x); v[2 * i + 1] = static_cast<float>(h.y);
    }
  }
  static __device__ __forceinline__ void load(const T* p, bool vec, float (&v)[8]) {
    if (vec) {
      open(raw(p), v);
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = static_cast<float>(p[i]);
    }
  }
  static __device__ __forceinline__ void store(T* p, bool vec, const float (&v)[8]) {
    if (vec) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; i++) w[i] = kv8_pack2<T>(v[2 * i], v[2 * i + 1]);
      *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; i++) p[i] = from(v[i]);
    }
  }
  static __device__ __forceinline__ T from(float x) { return T(x); }
};
template <> struct Elems<__half> : Elems16<__half, __half2> {};
template <> struct Elems<__nv_bfloat16> : Elems16<__nv_bfloat16, __nv_bfloat162> {};
#endif  // __CUDACC__

}  // namespace msb
