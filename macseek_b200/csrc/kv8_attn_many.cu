// Attention over the 8-bit cache (kv8_attn.cuh) for many query rows: chunks of prompts, whole prompts, large groups.
//
// Two products a tile of 128 keys, both on tcgen05 with halves and fp32 sums: S = Q K^T, operands in shared memory, and O += P V, the
// weights P taken from tensor memory, where they replace S.  The cache's codes become halves on the way into shared memory (exact); keys
// and values have one layout there, rows of 64 dims with the 128-byte swizzle: K-major for S, and for O read along the tokens.
//   warps     0..3, 4..7 a row tile of 128 each: a thread has a row, computes its weights and, when their reference moves, rescales O;
//             then four that convert keys and values, two buffers each; then one that issues the products.  While one row tile's weights
//             are computed the tensor core has the other's products.
//   F32 rows  queries and weights are two halves each: one row tile, and twice the products
//   TMEM      [0, 256): S (and P) of the row tiles, [256, 512): O; F32: [128, 192) the weights' second halves
// Bound by the exponentials, 16 a clock, beside the tensor core: 128 x 128 weights take as long as their two products of 128 dims.
// Every wait is bounded.
#include <algorithm>
#include "kv8_attn.cuh"
#include "ts_gemm.cuh"

namespace msb {

constexpr int kKmKeys = 128, kKmRows = 128;      // (kKmStep in kv8_attn.cu)

template <class T, int D>
struct KmShape {
  static constexpr bool kTwo = sizeof(T) == 4;
  static constexpr int kTiles = kTwo ? 1 : 2, kTerms = kTwo ? 2 : 1;
  static constexpr int kSoft = 4 * kTiles, kWarps = kSoft + 5;
  static constexpr int kBytes = 128 * D * 2;                          // a tile of 128 rows as halves
  static constexpr int kSmem = 2048 + kTiles * kTerms * kBytes + 4 * kBytes;
  static constexpr uint32_t kO = 256, kLow = 128;
};
struct KmHead {
  uint64_t kfull[2], kempty[2], vfull[2], vempty[2], sfull[2], pfull[2], ofull[2], qfull;
  uint32_t tmem_base;
  int abort_flag;
  float4 sc[2][kKmKeys / 16];       // key scale, exponent of the value scale, its inverse; of 16 tokens of a tile
};
static_assert(sizeof(KmHead) <= 1024, "the tiles follow");

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

template <class T, int D>
__global__ void __launch_bounds__(KmShape<T, D>::kWarps * 32, 1) kv8_attn_many_kernel(const Kv8AttnParams p) {
  using S = KmShape<T, D>;
  constexpr bool TWO = S::kTwo;
  extern __shared__ __align__(1024) uint8_t km_smem_raw[];
  uint8_t* smem = km_smem_raw + ((1024u - (smem_u32(km_smem_raw) & 1023u)) & 1023u);
  KmHead* hd = reinterpret_cast<KmHead*>(smem);
  uint8_t* qs_mem = smem + 1024;                                       // [tiles][terms][kBytes]
  uint8_t* kmem = qs_mem + S::kTiles * S::kTerms * S::kBytes;          // [2][kBytes]
  uint8_t* vmem = kmem + 2 * S::kBytes;
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
    for (int s = 0; s < 2; s++) {
      mbar_init(&hd->kfull[s], 4); mbar_init(&hd->kempty[s], 1); mbar_init(&hd->vfull[s], 4); mbar_init(&hd->vempty[s], 1);
      mbar_init(&hd->sfull[s], 1); mbar_init(&hd->pfull[s], 4); mbar_init(&hd->ofull[s], 1);
    }
    mbar_init(&hd->qfull, 4 * nt);
    hd->abort_flag = 0;
    mbar_fence_init();
  }
  if (warp == S::kWarps - 1) {
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

  if (warp == S::kWarps - 1) {
    // ------------------------------------------------------------------ products
    constexpr uint32_t base = (1u << 4) | ((uint32_t)(kKmRows >> 4) << 24);
    constexpr uint32_t is = base | ((uint32_t)(kKmKeys >> 3) << 17), io = base | (1u << 16) | ((uint32_t)(D >> 3) << 17);
    const bool leader = elect_one();
    const uint32_t q_s = smem_u32(qs_mem), k_s = smem_u32(kmem), v_s = smem_u32(vmem);
    auto scores = [&](int t, int s) {
#pragma unroll
      for (int e = 0; e < S::kTerms; e++)
#pragma unroll
        for (int k = 0; k < D / 16; k++) {
          const uint32_t o = (k >> 2) * 16384 + (k & 3) * 32;
          km_mma_ss(tmem + t * 128, ts_desc(q_s + (t * S::kTerms + e) * S::kBytes + o), ts_desc(k_s + s * S::kBytes + o), is, (e | k) ? 1u : 0u);
        }
      ts_commit(&hd->sfull[t]);
    };
    bool ok = wait(&hd->qfull, 0, kDevWaitFull) && wait(&hd->kfull[0], 0, kDevWaitFull);
    if (ok) {
      ts_fence_after();
      if (leader) {
        for (int t = 0; t < nt; t++) scores(t, 0);
        ts_commit(&hd->kempty[0]);
      }
      __syncwarp();
    }
    for (int j = 0; ok && j < n; j++) {
      const int s = j & 1;
      ok = wait(&hd->vfull[s], j >> 1, kDevWaitFull);
      for (int t = 0; ok && t < nt; t++) {
        ok = wait(&hd->pfull[t], j, kDevWaitFull) && (t || j + 1 >= n || wait(&hd->kfull[s ^ 1], (j + 1) >> 1, kDevWaitFull));
        if (!ok) break;
        ts_fence_after();
        if (leader) {
#pragma unroll
          for (int e = 0; e < S::kTerms; e++)
#pragma unroll
            for (int k = 0; k < kKmKeys / 16; k++)
              ts_mma_f16(tmem + S::kO + t * D, tmem + (e ? S::kLow : t * 128) + k * 8, km_desc_mn(v_s + s * S::kBytes + k * 2048, 16384), io,
                         (j | e | k) ? 1u : 0u);
          if (j + 1 < n) scores(t, s ^ 1);
          else ts_commit(&hd->ofull[t]);
        }
        __syncwarp();
      }
      if (ok && leader) {
        ts_commit(&hd->vempty[s]);
        if (j + 1 < n) ts_commit(&hd->kempty[s ^ 1]);
      }
      __syncwarp();
    }
  } else if (warp >= S::kSoft) {
    // ------------------------------------------------------------------ codes -> halves
    constexpr int kPer = D / 16;                       // 16-byte pieces a thread has of a tile
    const int c = tid - S::kSoft * 32, pc = c % (D / 16), row0 = c / (D / 16);
    const int* table = p.b.table + (size_t)blockIdx.y * p.b.table_stride;
    const int mask = (1 << p.c.shift) - 1;
    int ids = -1;
    auto look_up = [&](int j) {
      const int key = k0 + kKmKeys * j + 16 * lane;
      ids = -1;
      if (lane < kKmKeys / 16 && key < k1) {
        ids = __ldg(table + (key >> p.c.shift));
        if (ids < 0 || ids >= p.c.n_blocks) { ids = -1; atomicCAS(p.status, 0, kDevBadBatch); }
      }
    };
    uint4 r[kPer];
    auto load = [&](const uint8_t* codes, int j) {
#pragma unroll
      for (int i = 0; i < kPer; i++) {
        const int row = row0 + i * (128 / kPer), key = k0 + kKmKeys * j + row;
        const int id = __shfl_sync(0xffffffffu, ids, row >> 4);
        r[i] = make_uint4(0, 0, 0, 0);
        if (id >= 0 && key < sq.len)                   // rows behind the last token hold anything
          r[i] = __ldg(reinterpret_cast<const uint4*>(codes + ((((size_t)id * p.c.heads + kvh) << p.c.shift) + (key & mask)) * D) + pc);
      }
    };
    auto put = [&](uint8_t* dst) {
#pragma unroll
      for (int i = 0; i < kPer; i++) {
        const int row = row0 + i * (128 / kPer), j0 = 2 * (pc & 3), odd = pc >> 2;       // D 128: the upper half's lanes begin with the odd chunk
        const uint4 lo = make_uint4(kv8_half2(r[i].x), kv8_half2(r[i].x >> 16), kv8_half2(r[i].y), kv8_half2(r[i].y >> 16));
        const uint4 hi = make_uint4(kv8_half2(r[i].z), kv8_half2(r[i].z >> 16), kv8_half2(r[i].w), kv8_half2(r[i].w >> 16));
        uint8_t* q = dst + (pc >> 2) * 16384;
        *reinterpret_cast<uint4*>(q + km_at(row, j0 + odd)) = odd ? hi : lo;
        *reinterpret_cast<uint4*>(q + km_at(row, j0 + 1 - odd)) = odd ? lo : hi;
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
    };
    look_up(0);
    load(p.c.k, 0);
    for (int j = 0; j < n; j++) {
      const int s = j & 1;
      if (!wait(&hd->kempty[s], (j >> 1) ^ 1, kDevWaitEmpty)) break;
      put(kmem + s * S::kBytes);
      if (lane == 0) mbar_arrive(&hd->kfull[s]);
      load(p.c.v, j);
      float4 f = make_float4(0.f, -INFINITY, 0.f, 0.f);
      if (warp == S::kSoft && ids >= 0) {
        f.x = __ldg(p.c.ks + (size_t)ids * p.c.heads + kvh);
        const int e = kv8_exp(__ldg(p.c.vs + (size_t)ids * p.c.heads + kvh));
        f.y = (float)e; f.z = kv8_pow2(-e);
      }
      if (!wait(&hd->vempty[s], (j >> 1) ^ 1, kDevWaitEmpty)) break;     // with it the scales of two tiles ago have been used
      if (warp == S::kSoft && lane < kKmKeys / 16) hd->sc[s][lane] = f;
      put(vmem + s * S::kBytes);
      if (lane == 0) mbar_arrive(&hd->vfull[s]);
      if (j + 1 < n) { look_up(j + 1); load(p.c.k, j + 1); }
    }
  } else if ((warp >> 2) < nt) {
    // ------------------------------------------------------------------ weights: a row a thread
    const int t = warp >> 2, tr = tid & 127, row = m0 + t * kKmRows + tr;
    const bool live = row < R;
    const int tok = min(row, R - 1) / p.G, head = kvh * p.G + min(row, R - 1) % p.G, pos = sq.len - sq.n + tok;
    const int w0 = m0 + t * kKmRows + (warp & 3) * 32, w1 = min(w0 + 31, R - 1);
    const int all_hi = min(k1, sq.len - sq.n + min(w0, R - 1) / p.G + 1), all_lo = p.window ? sq.len - sq.n + w1 / p.G - p.window + 1 : 0;
    float f0;                                          // logit in binary exponents = product * f0 * key scale
    {
      const T* src = static_cast<const T*>(p.q) + (sq.row + tok) * p.q_stride + (int64_t)head * D;
      float top = 0.f, v[8];
#pragma unroll 4
      for (int c = 0; c < D / 8; c++) {
        Elems<T>::load(src + 8 * c, p.q_vec, v);
#pragma unroll
        for (int i = 0; i < 8; i++) top = fmaxf(top, fabsf(v[i]));
      }
      const int e = min(max((int)(__float_as_uint(top) >> 23) - 127, -60), 120);
      const float inv = p.scale < 0.f ? -kv8_pow2(-e) : kv8_pow2(-e);
      f0 = kv8_pow2(e) * fabsf(p.scale) * kLog2e;
      uint8_t* dst = qs_mem + t * S::kTerms * S::kBytes;
#pragma unroll 4
      for (int c = 0; c < D / 8; c++) {
        Elems<T>::load(src + 8 * c, p.q_vec, v);
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float a = live ? v[2 * i] * inv : 0.f, b = live ? v[2 * i + 1] * inv : 0.f;
          hi[i] = km_pack(a, b);
          if (TWO) {
            const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi[i]));
            lo[i] = km_pack(a - h.x, b - h.y);
          }
        }
        uint8_t* q = dst + (c >> 3) * 16384 + km_at(tr, c & 7);
        *reinterpret_cast<uint4*>(q) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        if (TWO) *reinterpret_cast<uint4*>(q + S::kBytes) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&hd->qfull);
    }
    const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16, ts = tmem + lanes + t * 128, to = tmem + lanes + S::kO + t * D;
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = 0; j < n; j++) {
      const int s = j & 1, base = k0 + kKmKeys * j;
      ok = wait(&hd->sfull[t], j, kDevWaitFull) && wait(&hd->vfull[s], j >> 1, kDevWaitFull);
      if (!ok) break;
      __syncwarp();
      ts_fence_after();
      const bool cut = base + kKmKeys > all_hi || base < all_lo;
      auto seen = [&](int col) {
        const int key = base + col;
        return key < k1 && key <= pos && (!p.window || key > pos - p.window);
      };
      uint32_t a[2][16];
      // ---- the largest exponent
      float top = -INFINITY;
      ts_ld16(ts, a[0]);
#pragma unroll
      for (int c = 0; c < kKmKeys / 16; c++) {
        ts_wait_ld();
        if (c + 1 < kKmKeys / 16) ts_ld16(ts + 16 * (c + 1), a[(c + 1) & 1]);
        const float4 sc = hd->sc[s][c];
        const float f = f0 * sc.x;
        float x = -INFINITY;
        if (cut) {
#pragma unroll
          for (int i = 0; i < 16; i++)
            if (seen(16 * c + i)) x = fmaxf(x, fmaf(__uint_as_float(a[c & 1][i]), f, sc.y));
        } else {
#pragma unroll
          for (int i = 0; i < 16; i++) x = fmaxf(x, __uint_as_float(a[c & 1][i]));
          x = fmaf(x, f, sc.y);
        }
        top = fmaxf(top, x);
        __syncwarp();
      }
      if (__any_sync(0xffffffffu, top > m + 8.f)) {
        const float nm = top > m + 8.f ? top : m, f = nm == -INFINITY ? 1.f : km_exp2(m - nm);
        m = nm; l *= f;
        if (j) {
#pragma unroll 1
          for (int c = 0; c < D / 16; c++) {
            ts_ld16(to + 16 * c, a[0]);
            ts_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; i++) a[0][i] = __float_as_uint(__uint_as_float(a[0][i]) * f);
            ts_st16(to + 16 * c, a[0]);
          }
        }
      }
      const float mm = m == -INFINITY ? 0.f : m;
      // ---- weights, in place of the products
      ts_ld16(ts, a[0]);
#pragma unroll
      for (int c = 0; c < kKmKeys / 16; c += 2) {
        uint32_t hi[16], lo[16];
#pragma unroll
        for (int h = 0; h < 2; h++) {
          ts_wait_ld();
          if (c + h + 1 < kKmKeys / 16) ts_ld16(ts + 16 * (c + h + 1), a[(h + 1) & 1]);
          const float4 sc = hd->sc[s][c + h];
          const float f = f0 * sc.x, b = sc.y - mm;
          float w[16], sum = 0.f;
#pragma unroll
          for (int i = 0; i < 16; i++) w[i] = fmaf(__uint_as_float(a[h][i]), f, b);
          if (cut) {
#pragma unroll
            for (int i = 0; i < 16; i++)
              if (!seen(16 * (c + h) + i)) w[i] = -INFINITY;
            __syncwarp();
          }
#pragma unroll
          for (int i = 0; i < 16; i++) { w[i] = km_exp2(w[i]); sum += w[i]; }
          l = fmaf(sum, sc.z, l);
#pragma unroll
          for (int i = 0; i < 8; i++) {
            hi[8 * h + i] = km_pack(w[2 * i], w[2 * i + 1]);
            if (TWO) {
              const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&hi[8 * h + i]));
              lo[8 * h + i] = km_pack(w[2 * i] - x.x, w[2 * i + 1] - x.y);
            }
          }
        }
        // the products of columns below 16 c + 32 have been read: [8 c, 8 c + 16) are free
        ts_st16(ts + 8 * c, hi);
        if (TWO) ts_st16(tmem + lanes + S::kLow + 8 * c, lo);
      }
      ts_wait_st();
      ts_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&hd->pfull[t]);
    }
    if (ok) ok = wait(&hd->ofull[t], 0, kDevWaitFull);
    if (ok) {
      __syncwarp();
      ts_fence_after();
      const bool last = p.splits == 1;
      float mul = 1.f;
      if (last) {
        float sum = l;
        if (p.sinks) sum += km_exp2(p.sinks[head] * kLog2e - (m == -INFINITY ? 0.f : m));
        mul = sum > 0.f ? 1.f / sum : sum != sum ? sum : 0.f;
      }
      const size_t at = ((size_t)split * p.b.n_tokens + sq.row + tok) * p.heads + head;
      if (!last && live) *reinterpret_cast<float2*>(kv8_part_ml(p, D) + 2 * at) = make_float2(m, l);
#pragma unroll 1
      for (int c = 0; c < D / 16; c++) {
        uint32_t a[16];
        __syncwarp();
        ts_ld16(to + 16 * c, a);
        ts_wait_ld();
        if (live) {
#pragma unroll
          for (int h = 0; h < 2; h++) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = __uint_as_float(a[8 * h + i]) * mul;
            if (last) Elems<T>::store(static_cast<T*>(p.out) + (sq.row + tok) * p.out_stride + (int64_t)head * D + 16 * c + 8 * h, p.out_vec, v);
            else Elems<float>::store(p.part + at * D + 16 * c + 8 * h, true, v);
          }
        }
      }
    }
  }
  ts_fence_before();
  __syncthreads();
  if (warp == S::kWarps - 1) {
    ts_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

template <class T, int D>
static int launch_many(const Kv8AttnParams& p, int groups, cudaStream_t st, int dev) {
  using S = KmShape<T, D>;
  auto kern = kv8_attn_many_kernel<T, D>;
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
int kv8_many_rows(int elem_type) { return elem_type == F32 ? kKmRows : 2 * kKmRows; }
int kv8_attn_many(const Kv8AttnParams& p, int groups, int elem_type, int D, cudaStream_t st, int dev) {
  if (elem_type == F32) return D == 64 ? launch_many<float, 64>(p, groups, st, dev) : launch_many<float, 128>(p, groups, st, dev);
  if (elem_type == F16) return D == 64 ? launch_many<__half, 64>(p, groups, st, dev) : launch_many<__half, 128>(p, groups, st, dev);
  return D == 64 ? launch_many<__nv_bfloat16, 64>(p, groups, st, dev) : launch_many<__nv_bfloat16, 128>(p, groups, st, dev);
}

}  // namespace msb
