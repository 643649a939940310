// Attention over the 8-bit cache (kv8_attn.cuh) for many query rows: chunks of prompts, whole prompts, large groups.
//
// Two products a tile of 64 keys, both on tcgen05 with halves and fp32 sums: S = Q K^T, operands in shared memory, and O += P V, the
// weights P taken from tensor memory, where they replace S.  The cache's codes become halves on the way into shared memory (exact); keys
// and values have one layout there, columns of 64 dims with the 128-byte swizzle: K-major for S, and for O read along the tokens.
//   warps     0..3, 4..7 a row tile of 128 each: a thread has a row, computes its weights and, when their reference moves, rescales O;
//             then four that convert keys and values, four buffers each; then one that issues the products
//   S         has two buffers a row tile: the scores of a tile are there before the weights of the one before are done.  (One buffer of 128
//             keys reads the queries half as often: 375 us for the prompt below and 107 for the chunks, when two were 403 and 98.)
//   F32 rows  queries and weights are two halves each: one row tile, and twice the products
//   TMEM      [256 t, ..): S of row tile t twice (64 columns; P in the first 32, F32: its second halves in the others), O from 128 on; F32: the
//             products of the second halves have a sum of their own from 384 on
//   sums      the tensor core cuts off what a sum does not hold, so O is added to a sum elsewhere and begun anew every 1024 keys (F32: tensor memory
//             from 256 on) or 16384 (16 bits: the scratch), and F32 scores begin with the queries' second halves.  200K tokens with values
//             of one sign, error without: 1.1e-3
// Bound by the exponentials (16 a clock beside those on the multiply-add pipe) and by shared memory: the products read 48 KB a tile and row
// tile, the conversion writes 32 KB.  4096 tokens, 64 heads over 8 of 128, bf16: 407 us = 675 TFLOP/s, of which an eighth goes into a block's
// start and end; ragged chunks of up to 333 tokens, 32 heads over 4 of 64, behind up to 8192: 92 us.  Every wait is bounded.
#include <algorithm>
#include "kv8_attn.cuh"
#include "ts_gemm.cuh"

namespace msb {

constexpr float kKmFirst = 7.f, kKmLow = 2048.f;      // exponent of the largest weight at first; what the second halves of weights are taken times
constexpr int kKmKeys = kKv8ManyStep, kKmRows = 128, kKmStages = 4, kKmHeadBytes = 4096;

template <class T, int D>
struct KmShape {
  static constexpr bool kTwo = sizeof(T) == 4;
  static constexpr int kTiles = kTwo ? 1 : 2, kTerms = kTwo ? 2 : 1;
  static constexpr int kSoft = 4 * kTiles, kMma = kSoft + 4, kWarps = kMma + 1;
  static constexpr int kQ = kKmRows * D * 2, kKv = kKmKeys * D * 2;      // bytes of a row tile's queries (a term), of a tile's keys or values
  static constexpr int kSmem = 1024 + kKmHeadBytes + kTiles * kTerms * kQ + 2 * kKmStages * kKv;
  static constexpr uint32_t kO = 128, kSum = 256, kO2 = 384;       // (kO2: what the second halves of the weights add to O, times kKmLow)
  static constexpr int kFold = kTwo ? kKv8FoldF32 / kKmKeys : kKv8Fold / kKmKeys;      // tiles whose products the tensor core adds up
};
struct KmHead {
  uint64_t kfull[kKmStages], kempty[kKmStages], vfull[kKmStages], vempty[kKmStages];
  uint64_t sfull[2][2], pfull[2][2], odone[2], ofull[2], qfull;        // [row tile][buffer]; odone: after each tile but the last, ofull: after that
  uint32_t tmem_base;
  int abort_flag;
  float f0[2 * kKmRows];
  float2 kept[2 * kKmRows];                 // km_fold's
  float4 sc[kKmStages][kKmKeys / 16];       // key scale, exponent of the value scale, its inverse; of 16 tokens of a tile
};
static_assert(sizeof(KmHead) <= kKmHeadBytes, "the tiles follow");

// place of the 16 bytes `j` of row r, 64 halves a row: 8-row groups of 1024 bytes, 128-byte swizzle
__device__ __forceinline__ uint32_t km_at(int r, int j) { return (uint32_t)((r >> 3) * 1024 + (r & 7) * 128 + ((j ^ (r & 7)) << 4)); }
__device__ __forceinline__ void km_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
// values: 64-dim columns of tokens, read along the tokens; the next 64 dims `next` bytes on, the next 8 tokens 1024
__device__ __forceinline__ uint64_t km_desc_mn(uint32_t saddr, uint32_t next) {
  return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(next >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ uint32_t km_pack(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float km_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 2^x of two numbers on the fused multiply-add pipe: x = n + r, |r| <= 1/2, a polynomial of degree 4 in r (minimax by Remez exchange, 2^-18.5)
// and n into its exponent.  [-126, 127]; what is below is as good as 0, what is above is looked at again
__device__ __forceinline__ void km_exp2_fma(float& a, float& b) {
  const float big = 12582912.f;                        // 1.5 * 2^23: the sum's last bits are the nearest whole number
  const uint64_t x = kv8_two(fminf(fmaxf(a, -126.f), 127.f), fminf(fmaxf(b, -126.f), 127.f));
  const uint64_t t = kv8_add2(x, kv8_two(big, big)), r = kv8_fma2(kv8_add2(t, kv8_two(-big, -big)), kv8_two(-1.f, -1.f), x);
  uint64_t p = kv8_fma2(r, kv8_two(0.009570102207362652f, 0.009570102207362652f), kv8_two(0.05591785907745361f, 0.05591785907745361f));
  p = kv8_fma2(p, r, kv8_two(0.240247443318367f, 0.240247443318367f));
  p = kv8_fma2(p, r, kv8_two(0.6931217908859253f, 0.6931217908859253f));
  p = kv8_fma2(p, r, kv8_two(0.9999992847442627f, 0.9999992847442627f));
  float pa, pb, ta, tb;
  kv8_apart(p, pa, pb);
  kv8_apart(t, ta, tb);
  a = __uint_as_float(__float_as_uint(pa) + (__float_as_uint(ta) << 23));
  b = __uint_as_float(__float_as_uint(pb) + (__float_as_uint(tb) << 23));
}

// 16 numbers of what has been taken out of a row's O: tensor memory (F32), or the row's place of the scratch, where 16-bit rows' O leaves no room
template <bool TWO>
__device__ __forceinline__ void km_sum_load(uint32_t column, const float* place, bool live, uint32_t (&b)[16]) {
  if constexpr (TWO) {
    ts_ld16(column, b);                               // (the caller waits)
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const float4 v = live ? __ldcg(reinterpret_cast<const float4*>(place) + i) : make_float4(0.f, 0.f, 0.f, 0.f);
      b[4 * i] = __float_as_uint(v.x); b[4 * i + 1] = __float_as_uint(v.y); b[4 * i + 2] = __float_as_uint(v.z); b[4 * i + 3] = __float_as_uint(v.w);
    }
  }
}
// The tensor core cuts off what a sum does not hold, up to 2^-23 of it at every 16 keys and always towards zero.  So O begins anew from time to
// time, and what it held is added to a sum in 32 bits; the row's sum of weights with it.  kept: the reference of that sum, the sum of weights.
// (Not inlined: the loop that calls it has no registers to spare.)
template <class T, int D>
__device__ __noinline__ void km_fold(uint32_t o, uint32_t column, float* place, bool live, bool first, float2* kept, float m, float l) {
  constexpr bool TWO = KmShape<T, D>::kTwo;
  const float f = first ? 0.f : km_exp2(kept->x - (m == -INFINITY ? 0.f : m));
#pragma unroll 1
  for (int c = 0; c < D / 16; c++) {
    uint32_t a[16], b[16] = {};
    if (!first) km_sum_load<TWO>(column + 16 * c, place + 16 * c, live, b);
    __syncwarp();
    ts_ld16(o + 16 * c, a);
    ts_wait_ld();
#pragma unroll
    for (int i = 0; i < 16; i++) a[i] = __float_as_uint(fmaf(__uint_as_float(b[i]), f, __uint_as_float(a[i])));
    if constexpr (TWO) {
      ts_st16(column + 16 * c, a);
    } else if (live) {
#pragma unroll
      for (int i = 0; i < 4; i++)
        __stcg(reinterpret_cast<float4*>(place + 16 * c) + i, make_float4(__uint_as_float(a[4 * i]), __uint_as_float(a[4 * i + 1]),
                                                                          __uint_as_float(a[4 * i + 2]), __uint_as_float(a[4 * i + 3])));
    }
    __syncwarp();
  }
  if constexpr (TWO) ts_wait_st();
  *kept = make_float2(m, first ? l : fmaf(kept->y, f, l));
}

// FOLD: parts may have more than kFold tiles (a prompt of 4096 tokens, bf16: 403 us without it, 411 with it; a chunk of 512 behind 200K 2 %)
template <class T, int D, bool FOLD>
__global__ void __launch_bounds__(KmShape<T, D>::kWarps * 32, 1) kv8_attn_many_kernel(const Kv8AttnParams p) {
  using S = KmShape<T, D>;
  constexpr bool TWO = S::kTwo;
  extern __shared__ __align__(1024) uint8_t km_smem_raw[];
  uint8_t* smem = km_smem_raw + ((1024u - (smem_u32(km_smem_raw) & 1023u)) & 1023u);
  KmHead* hd = reinterpret_cast<KmHead*>(smem);
  uint8_t* qs_mem = smem + kKmHeadBytes;                                      // [tiles][terms][kQ]
  uint8_t* kmem = qs_mem + S::kTiles * S::kTerms * S::kQ;              // [stages][kKv]
  uint8_t* vmem = kmem + kKmStages * S::kKv;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_launch_dependents();
  pdl_wait();
  const int kvh = blockIdx.x % p.c.heads, split = blockIdx.x / p.c.heads;
  const int m0 = (gridDim.z - 1 - blockIdx.z) * p.tile;                // the rows that see most keys first
  const Kv8Seq sq = kv8_seq(p.b, blockIdx.y, p.status);
  const int R = sq.n * p.G;
  if (m0 >= R) return;
  const int m1 = min(m0 + p.tile, R), nt = (m1 - m0 + kKmRows - 1) / kKmRows;
  const Kv8Range kr = kv8_range(sq, m0, m1, p.G, p.window, kKmKeys);
  const int k0 = kr.lo + split * p.chunk, k1 = min(kr.hi, k0 + p.chunk);
  if (k0 >= k1) return;
  const int n = (k1 - k0 + kKmKeys - 1) / kKmKeys;
  if (tid == 0) {
    for (int s = 0; s < kKmStages; s++) {
      mbar_init(&hd->kfull[s], 4); mbar_init(&hd->kempty[s], 1); mbar_init(&hd->vfull[s], 4); mbar_init(&hd->vempty[s], 1);
    }
    for (int t = 0; t < 2; t++) {
      for (int s = 0; s < 2; s++) { mbar_init(&hd->sfull[t][s], 1); mbar_init(&hd->pfull[t][s], 4); }
      mbar_init(&hd->odone[t], 1); mbar_init(&hd->ofull[t], 1);
    }
    mbar_init(&hd->qfull, 4 * nt);
    hd->abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == S::kMma) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&hd->tmem_base)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  ts_fence_before();
  __syncthreads();
  ts_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, hd->tmem_base, 0);
  volatile int* abort_flag = &hd->abort_flag;
  auto wait = [&](uint64_t* bar, uint32_t phase, int code) {
    return __all_sync(0xffffffffu, mbar_wait(bar, phase & 1u, abort_flag, p.status, code)) != 0;
  };

  if (warp == S::kMma) {
    // ------------------------------------------------------------------ products
    constexpr uint32_t base = (1u << 4) | ((uint32_t)(kKmRows >> 4) << 24);
    constexpr uint32_t is = base | ((uint32_t)(kKmKeys >> 3) << 17), io = base | (1u << 16) | ((uint32_t)(D >> 3) << 17);
    const bool leader = elect_one();
    const uint64_t q_d = ts_desc(smem_u32(qs_mem)), k_d = ts_desc(smem_u32(kmem)), v_d = km_desc_mn(smem_u32(vmem), kKmKeys * 128);
    bool ok = wait(&hd->qfull, 0, kDevWaitFull);
    // round j: the scores of tile j + 1, then the output's products of tile j (the loops stay rolled: unrolled weights made the prompt three times
    // as long)
#pragma unroll 1
    for (int j = -1; ok && j < n; j++) {
      if (j + 1 < n) {
        const int s = (j + 1) % kKmStages, b = (j + 1) & 1;
        ok = wait(&hd->kfull[s], (j + 1) / kKmStages, kDevWaitFull);
        if (!ok) break;
        ts_fence_after();
        if (leader) {
#pragma unroll 1
          for (int t = 0; t < nt; t++) {
#pragma unroll
            for (int e = S::kTerms - 1; e >= 0; e--)
#pragma unroll
              for (int k = 0; k < D / 16; k++)
                km_mma_ss(tmem + t * 256 + b * kKmKeys, q_d + (uint32_t)((t * S::kTerms + e) * (S::kQ >> 4) + (k >> 2) * (16384 >> 4) + (k & 3) * 2),
                          k_d + (uint32_t)(s * (S::kKv >> 4) + (k >> 2) * (kKmKeys * 128 >> 4) + (k & 3) * 2), is, (e < S::kTerms - 1 || k) ? 1u : 0u);
            ts_commit(&hd->sfull[t][b]);
          }
          ts_commit(&hd->kempty[s]);
        }
        __syncwarp();
      }
      if (j < 0) continue;
      const int s = j % kKmStages, b = j & 1;
      ok = wait(&hd->vfull[s], j / kKmStages, kDevWaitFull);
#pragma unroll 1
      for (int t = 0; ok && t < nt; t++) {
        ok = wait(&hd->pfull[t][b], j >> 1, kDevWaitFull);
        if (!ok) break;
        ts_fence_after();
        if (leader) {
#pragma unroll
          for (int e = 0; e < S::kTerms; e++)
#pragma unroll
            for (int k = 0; k < kKmKeys / 16; k++)
              ts_mma_f16(tmem + (e ? S::kO2 : t * 256 + S::kO), tmem + t * 256 + b * kKmKeys + e * (kKmKeys / 2) + k * 8,
                         v_d + (uint32_t)(s * (S::kKv >> 4) + k * (2048 >> 4)), io, ((e || !FOLD ? j : j % S::kFold) | k) ? 1u : 0u);
          ts_commit(j + 1 < n ? &hd->odone[t] : &hd->ofull[t]);
        }
        __syncwarp();
      }
      if (ok && leader) ts_commit(&hd->vempty[s]);
      __syncwarp();
    }
  } else if (warp >= S::kSoft && warp < S::kMma) {
    // ------------------------------------------------------------------ codes -> halves
    constexpr int kPer = D / 16, kRows = 128 / kPer;   // 16-byte pieces a thread has of two tiles, kRows rows apart
    // a quarter of a warp has two rows' pieces of one 64-dim half: its stores meet no bank twice
    const int c = tid - S::kSoft * 32, pc = D == 128 ? (c & 3) | (c >> 1 & 4) : c & 3, row0 = D == 128 ? (c >> 2 & 1) | (c >> 4) << 1 : c >> 2;
    const int* table = p.b.table + (size_t)blockIdx.y * p.b.table_stride;
    const int mask = (1 << p.c.shift) - 1;
    const uint32_t at0 = (pc >> 2) * (kKmKeys * 128) + km_at(row0, 2 * (pc & 3)), at1 = (pc >> 2) * (kKmKeys * 128) + km_at(row0, 2 * (pc & 3) + 1);
    // blocks of 16 tokens a lane, of the two tiles being put and of the next two: every load has two tiles' time to arrive (nothing looks
    // at an id before it is used)
    constexpr int kNone = -2147483647 - 1;
    auto look_up = [&](int j) {
      const int key = k0 + 2 * kKmKeys * j + 16 * lane;
      return lane < 2 * kKmKeys / 16 && key < k1 && key + 16 > kr.first ? __ldg(table + (key >> p.c.shift)) : kNone;
    };
    // every load is made, from the first block where there is none and of rows behind the last token (which hold anything): without branches
    // between them they leave one after the other.  What is not there becomes zeros when it is put.
    uint32_t low[kPer];
#pragma unroll
    for (int i = 0; i < kPer; i++) low[i] = (uint32_t)(((k0 + row0 + i * kRows) & mask) * D + pc * 16);      // (128 keys a round)
    uint4 rk[kPer], rv[kPer];
    auto load = [&](uint4 (&r)[kPer], const uint8_t* codes, int ids) {
      // head of the block, in units of 1024 bytes (a block of a head is 1024 at least)
      const uint32_t head = (uint32_t)(((((uint64_t)max(ids, 0) * p.c.heads + kvh) << p.c.shift) * D) >> 10);
#pragma unroll
      for (int i = 0; i < kPer; i++) {
        const uint32_t h = __shfl_sync(0xffffffffu, head, (row0 + i * kRows) >> 4);
        r[i] = __ldg(reinterpret_cast<const uint4*>(codes + ((uint64_t)h << 10) + low[i]));
      }
    };
    auto put = [&](uint8_t* dst, uint4 (&r)[kPer], int half, int ids, int j) {
      const int rows = sq.len - (k0 + 2 * kKmKeys * j);
      if (rows < 2 * kKmKeys || __any_sync(0xffffffffu, lane < 2 * kKmKeys / 16 && ids < 0)) {
#pragma unroll
        for (int i = 0; i < kPer; i++) {
          const int row = row0 + i * kRows, id = __shfl_sync(0xffffffffu, ids, row >> 4);
          if (i / (kPer / 2) == half && (id < 0 || row >= rows)) r[i] = make_uint4(0, 0, 0, 0);
        }
      }
#pragma unroll
      for (int i = 0; i < kPer; i++) {
        if (i / (kPer / 2) != half) continue;
        const int o = (i % (kPer / 2)) * kRows * 128;
        *reinterpret_cast<uint4*>(dst + at0 + o) = make_uint4(kv8_half2(r[i].x), kv8_half2(r[i].x >> 16), kv8_half2(r[i].y), kv8_half2(r[i].y >> 16));
        *reinterpret_cast<uint4*>(dst + at1 + o) = make_uint4(kv8_half2(r[i].z), kv8_half2(r[i].z >> 16), kv8_half2(r[i].w), kv8_half2(r[i].w >> 16));
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
    };
    const bool scales = warp == S::kSoft;
    int ids = -1, next = look_up(0);
    float ks = 0.f, vs = 1.f;
    // round j: tiles 2 j and 2 j + 1 from registers into shared memory, the next two into the registers
    const int rounds = (n + 1) / 2;
    bool ok = true;
#pragma unroll 1
    for (int j = -1; ok && j < rounds; j++) {
      const bool more = j + 1 < rounds;
      if (j >= 0) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const int i = 2 * j + h, s = i % kKmStages;
          if (!ok || i >= n) break;
          ok = wait(&hd->kempty[s], (i / kKmStages) ^ 1, kDevWaitEmpty);
          if (!ok) break;
          put(kmem + s * S::kKv, rk, h, ids, j);
          if (lane == 0) mbar_arrive(&hd->kfull[s]);
        }
      }
      if (more) {
        if (next < 0 || next >= p.c.n_blocks) {
          if (next != kNone) atomicCAS(p.status, 0, kDevBadBatch);
          next = -1;
        }
        load(rk, p.c.k, next);
      }
      if (j >= 0) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
          const int i = 2 * j + h, s = i % kKmStages;
          if (!ok || i >= n) break;
          ok = wait(&hd->vempty[s], (i / kKmStages) ^ 1, kDevWaitEmpty);   // with it the scales of four tiles ago have been used
          if (!ok) break;
          if (scales && lane / (kKmKeys / 16) == h) {
            const int e = kv8_exp(vs);
            hd->sc[s][lane % (kKmKeys / 16)] = ids < 0 ? make_float4(0.f, -INFINITY, 0.f, 0.f) : make_float4(ks, (float)e, kv8_pow2(-e), 0.f);
          }
          put(vmem + s * S::kKv, rv, h, ids, j);
          if (lane == 0) mbar_arrive(&hd->vfull[s]);
        }
      }
      if (more) {
        load(rv, p.c.v, next);
        if (scales && next >= 0) {
          ks = __ldg(p.c.ks + (size_t)next * p.c.heads + kvh);
          vs = __ldg(p.c.vs + (size_t)next * p.c.heads + kvh);
        }
        ids = next;
        next = j + 2 < rounds ? look_up(j + 2) : kNone;
      }
    }
  } else if (warp < S::kSoft && (warp >> 2) < nt) {
    // ------------------------------------------------------------------ weights: a row a thread
    const int t = warp >> 2, tr = tid & 127, row = m0 + t * kKmRows + tr;
    const bool live = row < R;
    const int tok = min(row, R - 1) / p.G, head = kvh * p.G + min(row, R - 1) % p.G, pos = sq.len - sq.n + tok;
    const int w0 = m0 + t * kKmRows + (warp & 3) * 32, w1 = min(w0 + 31, R - 1);
    const int all_hi = min(k1, sq.len - sq.n + min(w0, R - 1) / p.G + 1), all_lo = p.window ? sq.len - sq.n + w1 / p.G - p.window + 1 : 0;
    {
      // the warp's 32 rows, D / 8 lanes a row: their largest, then halves.  A logit in binary exponents is product * f0 * key scale
      constexpr int kLanes = D / 8, kAtOnce = 32 / kLanes;
      uint8_t* dst = qs_mem + t * S::kTerms * S::kQ;
      const int c = lane % kLanes, dq = kAtOnce / p.G, dr = kAtOnce % p.G;
      constexpr int kBatch = TWO ? 4 : 8;              // rows requested at once
      int rr = w0 + lane / kLanes, tk = rr / p.G, hh = rr - tk * p.G;        // row, token, head of the group
#pragma unroll 1
      for (int i0 = 0; i0 < kLanes; i0 += kBatch) {
        typename Elems<T>::Raw x[kBatch] = {};
        const T* src[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; i++) {
          src[i] = rr < R ? static_cast<const T*>(p.q) + (sq.row + tk) * p.q_stride + (kvh * p.G + hh) * D + 8 * c : nullptr;
          rr += kAtOnce; tk += dq; hh += dr;
          if (hh >= p.G) { hh -= p.G; tk++; }
          if (p.q_vec && src[i]) x[i] = Elems<T>::raw(src[i]);
        }
        if (!p.q_vec) {
#pragma unroll
          for (int i = 0; i < kBatch; i++) {
            T* y = reinterpret_cast<T*>(&x[i]);
            if (src[i])
#pragma unroll
              for (int k = 0; k < 8; k++) y[k] = src[i][k];
          }
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < kBatch; i++) {
          const int r = (i0 + i) * kAtOnce + lane / kLanes;
          float v[8], top = 0.f;
          Elems<T>::open(x[i], v);
#pragma unroll
          for (int k = 0; k < 8; k++) top = fmaxf(top, fabsf(v[k]));
#pragma unroll
          for (int o = kLanes / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          const int e = min(max((int)(__float_as_uint(top) >> 23) - 127, -126), 120);
          const float inv = p.scale < 0.f ? -kv8_pow2(-e) : kv8_pow2(-e);
          if (c == 0) hd->f0[t * 128 + (warp & 3) * 32 + r] = kv8_pow2(e) * fabsf(p.scale) * kLog2e;
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int k = 0; k < 4; k++) {
            hi[k] = km_pack(v[2 * k] * inv, v[2 * k + 1] * inv);
            if (TWO) {
              const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi[k]));
              lo[k] = km_pack(v[2 * k] * inv - h.x, v[2 * k + 1] * inv - h.y);
            }
          }
          uint8_t* q = dst + (c >> 3) * 16384 + km_at((warp & 3) * 32 + r, c & 7);
          *reinterpret_cast<uint4*>(q) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          if (TWO) *reinterpret_cast<uint4*>(q + S::kQ) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&hd->qfull);
    }
    const float f0 = hd->f0[t * 128 + tr];
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16, to = tmem + lanes + t * 256 + S::kO;
    const int first = p.window ? max(0, pos - p.window + 1) : 0, last = min(k1 - 1, pos);      // keys that the row sees
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j0 = 0, j1; ok && j0 < n; j0 = j1) {
      j1 = FOLD ? min(n, j0 + S::kFold) : n;
      if (FOLD && j0) {
        // (the scores of this tile first: with them the products of two tiles ago are there, and the phase waited for is the next)
        ok = wait(&hd->sfull[t][j0 & 1], j0 >> 1, kDevWaitFull) && wait(&hd->odone[t], j0 - 1, kDevWaitFull);
        if (!ok) break;
        __syncwarp();
        ts_fence_after();
        km_fold<T, D>(to, tmem + lanes + S::kSum, p.part + (((size_t)split * p.b.n_tokens + sq.row + tok) * p.heads + head) * D, live, j0 == S::kFold,
                      &hd->kept[t * 128 + tr], m, l);
        l = 0.f;
      }
#pragma unroll 1
      for (int j = j0; j < j1; j++) {
        const int s = j % kKmStages, base = k0 + kKmKeys * j;
        const uint32_t ts = tmem + lanes + t * 256 + (j & 1) * kKmKeys;
        ok = wait(&hd->sfull[t][j & 1], j >> 1, kDevWaitFull) && wait(&hd->vfull[s], j / kKmStages, kDevWaitFull);     // the scales come with the values
        if (!ok) break;
        __syncwarp();
        ts_fence_after();
        const bool cut = base + kKmKeys > all_hi || base < all_lo;
        float mm = m == -INFINITY ? 0.f : m;
        if (__any_sync(0xffffffffu, m == -INFINITY)) {   // no reference yet: the tile's largest exponent
          float top = -INFINITY;
#pragma unroll 1
          for (int c = 0; c < kKmKeys / 16; c++) {
            uint32_t a[16];
            ts_ld16(ts + 16 * c, a);
            ts_wait_ld();
            const float4 sc = hd->sc[s][c];
            const float f = f0 * sc.x;
            const int hi = cut ? last - base - 16 * c : 16, lo = cut ? first - base - 16 * c : 0;
#pragma unroll
            for (int i = 0; i < 16; i++)
              if (i <= hi && i >= lo) top = fmaxf(top, __fmaf_rd(__uint_as_float(a[i]), f, sc.y));
            __syncwarp();
          }
          if (m == -INFINITY) m = __fadd_rd(floorf(top), -kKmFirst);
          mm = m == -INFINITY ? 0.f : m;
        }
        // ---- weights.  The reference begins 7 below the first tile's largest exponent and stays unless the weights of 16 keys sum to more than
        // 60000 (a half holds each of them below that).  Then those of the warp's rows that sum to more than 2^8 move up by a whole number, to a
        // sum of 2^6 to 2^7, what has been summed against the old reference is scaled, and the weights are made again.  (Were only the row
        // above 60000 moved, a prompt of 4096 tokens takes 4 % longer.)
        // A half holds nothing below 2^-25, so N keys lose N 2^-31 at most beside the largest; the second halves of F32 weights, taken times
        // 2^11, hold what is 2^11 below
        bool lost = false;
        constexpr int kTries = 4;
        int tries = 0;
        uint32_t w[4][16];
        float part[4];
#pragma unroll 1
        for (;;) {
#pragma unroll
          for (int h = 0; h < 4; h++) ts_ld16(ts + 16 * h, w[h]);
          ts_wait_ld();
#pragma unroll
          for (int h = 0; h < 4; h++) {
            const float4 sc = hd->sc[s][h];
            const float off = __fadd_ru(sc.y, -mm);
            const uint64_t f = kv8_two(f0 * sc.x, f0 * sc.x), b = kv8_two(off, off);
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
              float x, y;
              kv8_apart(kv8_fma2(kv8_two(__uint_as_float(w[h][i]), __uint_as_float(w[h][i + 1])), f, b), x, y);
              w[h][i] = __float_as_uint(x); w[h][i + 1] = __float_as_uint(y);
            }
          }
          if (cut || tries == kTries) {
            const int hi = cut ? last - base : 64, lo = cut ? first - base : 0;
            const float most = tries == kTries && !lost ? 15.f : INFINITY;
#pragma unroll
            for (int i = 0; i < 64; i++) {
              float x;
              asm("min.NaN.f32 %0, %1, %2;" : "=f"(x) : "f"(__uint_as_float(w[i >> 4][i & 15])), "f"(most));
              w[i >> 4][i & 15] = i > hi || i < lo ? 0xFF800000u : __float_as_uint(x);
            }
            __syncwarp();
          }
#pragma unroll
          for (int h = 0; h < 4; h++) {
            uint64_t x[2] = {0, 0};
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
              float u = __uint_as_float(w[h][i]), v = __uint_as_float(w[h][i + 1]);
              if (!TWO && (i & 6) == 6) km_exp2_fma(u, v);       // a quarter of them beside the others (F32 keeps its two units' accuracy)
              else { u = km_exp2(u); v = km_exp2(v); }
              w[h][i] = __float_as_uint(u); w[h][i + 1] = __float_as_uint(v);
              x[i >> 1 & 1] = kv8_add2(x[i >> 1 & 1], kv8_two(u, v));
            }
            float y, z;
            kv8_apart(kv8_add2(x[0], x[1]), y, z);
            part[h] = y + z;
          }
          const float most = fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3]));
          if (tries == kTries || !__any_sync(0xffffffffu, most > 60000.f && !lost)) break;
          // by the next power of two above the sum, or, where that is beyond 32 bits or near the end of km_exp2_fma's range (which a sum then
          // does not show to be passed), to the largest exponent.  A row whose products are infinite has none.  The reference is a whole number;
          // beyond 2^27 not every one is held, and it is the next one down (weights come out larger, never smaller), and after four times weights
          // that are still too large become 2^15, all of them: their logits differ by less than a step of 32 bits
          constexpr float kFar = 100.f;
          float up = most > 256.f && !lost ? (float)((int)(__float_as_uint(most) >> 23) - 126) - kKmFirst : 0.f;
          if (__any_sync(0xffffffffu, up > kFar)) {
            float top = -INFINITY;
#pragma unroll 1
            for (int k = 0; k < 4; k++) {
              ts_ld16(ts + 16 * k, w[0]);
              ts_wait_ld();
              const float4 sc = hd->sc[s][k];
#pragma unroll
              for (int i = 0; i < 16; i++) {
                const int key = base + 16 * k + i;
                if (!cut || (key >= first && key <= last)) top = fmaxf(top, __fmaf_rd(__uint_as_float(w[0][i]), f0 * sc.x, __fadd_ru(sc.y, -mm)));
              }
              __syncwarp();
            }
            if (up > kFar) {
              lost = !(top < INFINITY);
              up = lost ? 0.f : ceilf(top) - kKmFirst;
            }
          }
          tries++;
          const float moved = up > 0.f ? __fadd_rd(m, up) : m, f = moved > m ? km_exp2(m - moved) : 1.f;
          if (moved > m) m = mm = moved;
          l *= f;
          if (j) {                                       // the products of the tile before are there (those of two before are: this tile's scores are)
            ok = wait(&hd->odone[t], j - 1, kDevWaitFull);
            if (!ok) break;
            __syncwarp();
            ts_fence_after();
#pragma unroll 1
            for (int k = 0; k < S::kTerms * (D / 16); k++) {
              const uint32_t at = k < D / 16 ? to + 16 * k : tmem + lanes + S::kO2 + 16 * (k - D / 16);
              ts_ld16(at, w[0]);
              ts_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; i++) w[0][i] = __float_as_uint(__uint_as_float(w[0][i]) * f);
              ts_st16(at, w[0]);
            }
            ts_wait_st();
          }
        }
        if (!ok) break;
#pragma unroll
        for (int h = 0; h < 4; h++) l = fmaf(part[h], hd->sc[s][h].z, l);
#pragma unroll
        for (int h = 0; h < 4; h += 2) {                 // in place of the products, all of which have been read
          uint32_t hi[16], lo[16];
#pragma unroll
          for (int i = 0; i < 16; i++) {
            const float u = __uint_as_float(w[h + (i >> 3)][2 * i & 15]), v = __uint_as_float(w[h + (i >> 3)][(2 * i & 15) + 1]);
            hi[i] = km_pack(u, v);
            if (TWO) {
              const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&hi[i]));
              lo[i] = km_pack((u - y.x) * kKmLow, (v - y.y) * kKmLow);
            }
          }
          ts_st16(ts + 8 * h, hi);
          if constexpr (TWO) ts_st16(ts + kKmKeys / 2 + 8 * h, lo);
        }
        ts_wait_st();
        ts_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&hd->pfull[t][j & 1]);
      }
    }
    ok = ok && wait(&hd->ofull[t], 0, kDevWaitFull);
    if (ok) {
      __syncwarp();
      ts_fence_after();
      const bool whole = p.splits == 1;
      const size_t at = ((size_t)split * p.b.n_tokens + sq.row + tok) * p.heads + head;
      float mul = 1.f, f_sum = 0.f;
      if (FOLD && n > S::kFold) {
        const float2 kept = hd->kept[t * 128 + tr];
        f_sum = km_exp2(kept.x - (m == -INFINITY ? 0.f : m));
        l = fmaf(kept.y, f_sum, l);
      }
      if (whole) {
        float sum = l;
        if (p.sinks) sum += km_exp2(p.sinks[head] * kLog2e - (m == -INFINITY ? 0.f : m));
        // (a row that sees nothing has no reference, and a sum only of what km_exp2_fma makes of its -infinities)
        mul = sum != sum ? sum : m > -INFINITY && sum > 0.f ? 1.f / sum : 0.f;
      } else if (live) {
        *reinterpret_cast<float2*>(kv8_part_ml(p, D) + 2 * at) = make_float2(m, l);
      }
      // a row to the place of its queries (which nothing reads any more), then whole rows at a time to memory
      constexpr int kRowBytes = D * sizeof(T), kPieces = kRowBytes / 16;
      uint8_t* rows = qs_mem + (t * kKmRows + (warp & 3) * 32) * kRowBytes;
#pragma unroll 1
      for (int c = 0; c < D / 16; c++) {
        uint32_t a[16];
        __syncwarp();
        ts_ld16(to + 16 * c, a);
        ts_wait_ld();
        if (TWO) {
          uint32_t b[16];
          ts_ld16(tmem + lanes + S::kO2 + 16 * c, b);
          ts_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; i++) a[i] = __float_as_uint(fmaf(__uint_as_float(b[i]), 1.f / kKmLow, __uint_as_float(a[i])));
        }
        if (FOLD && n > S::kFold) {
          uint32_t b[16];
          km_sum_load<TWO>(tmem + lanes + S::kSum + 16 * c, p.part + at * D + 16 * c, live, b);
          ts_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; i++) a[i] = __float_as_uint(fmaf(__uint_as_float(b[i]), f_sum, __uint_as_float(a[i])));
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
          float v[8];
#pragma unroll
          for (int i = 0; i < 8; i++) v[i] = __uint_as_float(a[8 * h + i]) * mul;
          if (whole) {
            const int o = (2 * c + h) * (8 * sizeof(T) / 16);
#pragma unroll
            for (int k = 0; k < (int)(8 * sizeof(T) / 16); k++)
              *reinterpret_cast<uint4*>(rows + lane * kRowBytes + (((o + k) ^ (lane & 7)) << 4)) = Elems<T>::pack16(v, k);
          } else if (live) {
            Elems<float>::store(p.part + at * D + 16 * c + 8 * h, true, v);
          }
        }
      }
      if (whole) {
        __syncwarp();
        const int64_t mine = (sq.row + tok) * p.out_stride + (int64_t)head * D;
#pragma unroll 4
        for (int i = 0; i < kPieces; i++) {            // 32 pieces of the warp's 32 rows at a time
          const int c = i * 32 + lane, r = c / kPieces, pc = c % kPieces;
          const int64_t o = __shfl_sync(0xffffffffu, mine, r);
          if (w0 + r < R) {
            T* dst = static_cast<T*>(p.out) + o + pc * (16 / (int)sizeof(T));
            const uint4 u = *reinterpret_cast<const uint4*>(rows + r * kRowBytes + ((pc ^ (r & 7)) << 4));
            if (p.out_vec) {
              *reinterpret_cast<uint4*>(dst) = u;
            } else {
              const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
              for (int k = 0; k < (int)(16 / sizeof(T)); k++) dst[k] = e[k];
            }
          }
          __syncwarp();
        }
      }
    }
  }
  ts_fence_before();
  __syncthreads();
  if (warp == S::kMma) {
    ts_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

template <class T, int D, bool FOLD>
static int launch_many(const Kv8AttnParams& p, int groups, cudaStream_t st, int dev) {
  using S = KmShape<T, D>;
  auto kern = kv8_attn_many_kernel<T, D, FOLD>;
  const int smem = std::max(S::kSmem, 120 * 1024);       // one block an SM: it takes the whole tensor memory
  static bool done[64] = {};
  if (!done[dev & 63]) {
    MSB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    done[dev & 63] = true;
  }
  MSB_CUDA(launch_pdl(kern, dim3(p.c.heads * p.splits, p.b.n_seq, groups), dim3(S::kWarps * 32), (size_t)smem, st, p));
  MSB_LAUNCH_CHECK("kv8_attn");
  return kOk;
}
static_assert(kKv8ManyRowsF32 == kKmRows && kKv8ManyRows == 2 * kKmRows, "row tiles of a block");
int kv8_attn_many(const Kv8AttnParams& p, int groups, int elem_type, int D, cudaStream_t st, int dev) {
  const bool fold = p.chunk > kKv8Fold;
#define KM_GO(T, FOLD) return D == 64 ? launch_many<T, 64, FOLD>(p, groups, st, dev) : launch_many<T, 128, FOLD>(p, groups, st, dev)
  if (elem_type == F32) KM_GO(float, true);
  if (elem_type == F16) { if (fold) KM_GO(__half, true); KM_GO(__half, false); }
  if (fold) KM_GO(__nv_bfloat16, true);
  KM_GO(__nv_bfloat16, false);
#undef KM_GO
}

}  // namespace msb
