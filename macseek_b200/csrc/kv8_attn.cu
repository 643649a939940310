// Attention over the 8-bit cache (kv8_attn.cuh) for few query rows: single tokens and short drafts.
//
// Every code is read once and what bounds the kernel is that read.  A block of four warps takes 16 rows of one key head (mma.sync
// m16n8k16: a whole group of query heads, several tokens of a draft) over one range of keys; a warp takes every fourth step of 16 tokens.
// Steps are fetched by the warp itself, with cp.async into its own ring, so that the warps never wait for one another before the end.
//   scores   the contraction may run over the dims in any order: a lane takes 16 neighbouring bytes of "its" token as eight pairs and
//            the query's registers are laid out alike; a pair of codes is one conversion to two halves (exact)
//   output   the tokens are contracted: bytes of two neighbouring tokens are interleaved and converted; lane g holds dims [16 g, 16 g + 16)
// The queries are scaled by a power of two to at most 2 in a row and used as halves; F32 ones, and their weights, as two halves each.
#include <algorithm>
#include "kv8_attn.cuh"

namespace msb {

constexpr int kKdWarps = 4, kKdStages = 4, kKdStep = 16, kKdRows = 16;

__device__ __forceinline__ void kd_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 16 bytes, zeros where !there
__device__ __forceinline__ void kd_copy16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ uint32_t kd_pack(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <bool TWO>
__device__ __forceinline__ void kd_split(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = kd_pack(a, b);
  if (TWO) {
    const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    lo = kd_pack(a - h.x, b - h.y);
  }
}
__device__ __forceinline__ float kd_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <int D>
struct KdTile {
  static constexpr int kBytes = kKdStep * D;
  // where 16-byte chunk c of row r lies.  D 128: the keys' reads (rows r, r + 1; chunks t, t + 4) and the values' (rows 2 t, chunks g) are
  // free of bank conflicts with these; D 64: rows 4..7 and 12..15 change places in pairs as well
  static __device__ __forceinline__ uint32_t key(int r, int c) { return D == 128 ? r * 128 + ((c ^ ((r & 1) << 2)) << 4) : r * 64 + (c << 4); }
  static __device__ __forceinline__ uint32_t val(int r, int c) {
    return D == 128 ? r * 128 + ((c ^ (r & 6)) << 4) : (r ^ ((r >> 2) & 1)) * 64 + ((c ^ (((r >> 1) & 1) << 1)) << 4);
  }
};

template <class T, int D>
__global__ void __launch_bounds__(kKdWarps * 32, 3) kv8_attn_few_kernel(const Kv8AttnParams p) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr bool TWO = sizeof(T) == 4;
  constexpr int KS = D / 16, NT = D / 8, CH = D / 64;      // k-steps, output tiles, 16-byte chunks of a key row per lane
  constexpr int kWarpBytes = kKdStages * 2 * KdTile<D>::kBytes, kPitch = D + 4;
  extern __shared__ __align__(16) uint8_t kd_smem[];
  __shared__ float s_m[kKdWarps][kKdRows], s_l[kKdWarps][kKdRows];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int tiles = gridDim.y / p.c.heads, kvh = blockIdx.y / tiles, m0 = (blockIdx.y % tiles) * kKdRows;
  const Kv8Seq sq = kv8_seq(p.b, blockIdx.z, p.status);
  const int R = sq.n * p.G;
  if (m0 >= R) return;
  const int m1 = min(m0 + kKdRows, R);
  const Kv8Range kr = kv8_range(sq, m0, m1, p.G, p.window, kKdStep);
  const int k0 = kr.lo + blockIdx.x * p.chunk, k1 = min(kr.hi, k0 + p.chunk);
  if (k0 >= k1) return;
  const int steps = (k1 - k0 + kKdStep - 1) / kKdStep;
  const int mine = steps > warp ? (steps - warp + kKdWarps - 1) / kKdWarps : 0;
  const int* table = p.b.table + (size_t)blockIdx.z * p.b.table_stride;
  const uint32_t ring = smem_u32(kd_smem) + warp * kWarpBytes;

  // ---- block ids and scales of the warp's next 32 steps, one step per lane
  int ids = -1;
  float ksc = 0.f, vex = 0.f;
  auto look_up = [&](int i) {
    const int step = warp + kKdWarps * (i + lane);
    ids = -1; ksc = 0.f; vex = 0.f;
    if (step < steps) {
      ids = __ldg(table + ((k0 + kKdStep * step) >> p.c.shift));
      if (ids < 0 || ids >= p.c.n_blocks) { ids = -1; atomicCAS(p.status, 0, kDevBadBatch); }
      else {
        ksc = __ldg(p.c.ks + (size_t)ids * p.c.heads + kvh);
        vex = (float)kv8_exp(__ldg(p.c.vs + (size_t)ids * p.c.heads + kvh));
      }
    }
  };
  auto fetch = [&](int i) {                   // step i of the warp; its lane's ids are loaded
    if (i < mine) {
      const int id = __shfl_sync(0xffffffffu, ids, i & 31);
      const int base = k0 + kKdStep * (warp + kKdWarps * i);
      const size_t off = ((((size_t)max(id, 0) * p.c.heads + kvh) << p.c.shift) + (base & ((1 << p.c.shift) - 1))) * D;
      const uint32_t dst = ring + (i % kKdStages) * 2 * KdTile<D>::kBytes;
#pragma unroll
      for (int j = 0; j < D / 32; j++) {
        const int c = lane + 32 * j, r = c / (D / 16), ch = c % (D / 16);
        const bool there = id >= 0 && base + r < sq.len;     // rows behind the last token hold anything
        kd_copy16(dst + KdTile<D>::key(r, ch), p.c.k + off + c * 16, there);
        kd_copy16(dst + KdTile<D>::kBytes + KdTile<D>::val(r, ch), p.c.v + off + c * 16, there);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  look_up(0);
  float ks_cur = ksc, ve_cur = vex;           // of the batch that is being computed (the fetches run ahead into the next one)
  int id_cur = ids;
#pragma unroll
  for (int i = 0; i < kKdStages - 1; i++) fetch(i);

  // ---- queries: rows g and g + 8 of the tile, scaled to at most 2
  uint32_t qh[KS][4], ql[TWO ? KS : 1][4];
  float qs[2];
  int qpos[2];
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const int r = m0 + g + 8 * h, tok = min(r, R - 1) / p.G, head = kvh * p.G + min(r, R - 1) % p.G;
    const T* src = static_cast<const T*>(p.q) + (sq.row + tok) * p.q_stride + (int64_t)head * D;
    qpos[h] = r < R ? sq.len - sq.n + tok : -1;              // a row that is not there sees nothing
    float v[CH][16];
    float top = 0.f;
#pragma unroll
    for (int j = 0; j < CH; j++) {
      float a[8];
#pragma unroll
      for (int e = 0; e < 2; e++) {
        Elems<T>::load(src + 16 * (t + 4 * j) + 8 * e, p.q_vec, a);
#pragma unroll
        for (int i = 0; i < 8; i++) { v[j][8 * e + i] = a[i]; top = fmaxf(top, fabsf(a[i])); }
      }
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int e = min(max((int)(__float_as_uint(top) >> 23) - 127, -100), 120);
    const float inv = kv8_pow2(-e);
    qs[h] = kv8_pow2(e) * p.scale * kLog2e;
#pragma unroll
    for (int j = 0; j < CH; j++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        uint32_t lo[2];
        kd_split<TWO>(v[j][4 * i] * inv, v[j][4 * i + 1] * inv, qh[4 * j + i][h], lo[0]);
        kd_split<TWO>(v[j][4 * i + 2] * inv, v[j][4 * i + 3] * inv, qh[4 * j + i][2 + h], lo[1]);
        if (TWO) { ql[4 * j + i][h] = lo[0]; ql[4 * j + i][2 + h] = lo[1]; }
      }
  }

  float o[NT][4];
#pragma unroll
  for (int i = 0; i < NT; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  const uint8_t* kbase = kd_smem + warp * kWarpBytes;

  for (int i = 0; i < mine; i++) {
    if (i + kKdStages - 1 < mine && ((i + kKdStages - 1) & 31) == 0) look_up(i + kKdStages - 1);
    fetch(i + kKdStages - 1);
    if (i && (i & 31) == 0) { ks_cur = ksc; ve_cur = vex; id_cur = ids; }
    asm volatile("cp.async.wait_group %0;" ::"n"(kKdStages - 1) : "memory");
    __syncwarp();
    const uint8_t* kt = kbase + (i % kKdStages) * 2 * KdTile<D>::kBytes;
    const uint8_t* vt = kt + KdTile<D>::kBytes;
    const int base = k0 + kKdStep * (warp + kKdWarps * i);
    const float ks = __shfl_sync(0xffffffffu, ks_cur, i & 31), ve = __shfl_sync(0xffffffffu, ve_cur, i & 31);
    const bool ok = __shfl_sync(0xffffffffu, id_cur, i & 31) >= 0;
    // ---- scores of 16 tokens
    float s[2][4];
#pragma unroll
    for (int nt = 0; nt < 2; nt++) {
      s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
      for (int j = 0; j < CH; j++) {
        const uint4 u = *reinterpret_cast<const uint4*>(kt + KdTile<D>::key(8 * nt + g, t + 4 * j));
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int x = 0; x < 4; x++) {
          const uint32_t b0 = kv8_half2(w[x]), b1 = kv8_half2(w[x] >> 16);
          kd_mma(s[nt], qh[4 * j + x], b0, b1);
          if (TWO) kd_mma(s[nt], ql[4 * j + x], b0, b1);
        }
      }
    }
    // ---- weights
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const float f = qs[h] * ks;
#pragma unroll
      for (int nt = 0; nt < 2; nt++)
#pragma unroll
        for (int x = 0; x < 2; x++) {
          const int key = base + 8 * nt + 2 * t + x;
          const bool seen = ok && key < k1 && key <= qpos[h] && (!p.window || key > qpos[h] - p.window);
          float& v = s[nt][2 * h + x];
          v = seen ? fmaf(v, f, ve) : -INFINITY;
          top[h] = fmaxf(top[h], v);
        }
      top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
      top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
    }
    if (__any_sync(0xffffffffu, top[0] > m[0] || top[1] > m[1])) {
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const float n = fmaxf(m[h], top[h]), f = n == -INFINITY ? 1.f : kd_exp2(m[h] - n);
        m[h] = n; l[h] *= f;
#pragma unroll
        for (int k = 0; k < NT; k++) { o[k][2 * h] *= f; o[k][2 * h + 1] *= f; }
      }
    }
    const float vi = kv8_pow2(-(int)ve);
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const float mm = m[h] == -INFINITY ? 0.f : m[h];
      float sum = 0.f;
#pragma unroll
      for (int nt = 0; nt < 2; nt++)
#pragma unroll
        for (int x = 0; x < 2; x++) {
          float& v = s[nt][2 * h + x];
          v = kd_exp2(v - mm);
          sum += v;
        }
      l[h] = fmaf(sum, vi, l[h]);
    }
    uint32_t ph[4], pl[4];
    kd_split<TWO>(s[0][0], s[0][1], ph[0], pl[0]);
    kd_split<TWO>(s[0][2], s[0][3], ph[1], pl[1]);
    kd_split<TWO>(s[1][0], s[1][1], ph[2], pl[2]);
    kd_split<TWO>(s[1][2], s[1][3], ph[3], pl[3]);
    // ---- output: lane g has dims [g D / 8, (g + 1) D / 8), tile j its j-th
    uint32_t x[4][NT / 4];
#pragma unroll
    for (int r = 0; r < 4; r++) {
      const int row = 2 * t + (r & 1) + 8 * (r >> 1);
      if (D == 128) {
        const uint4 u = *reinterpret_cast<const uint4*>(vt + KdTile<D>::val(row, g));
        x[r][0] = u.x; x[r][1] = u.y; x[r][NT / 4 - 2] = u.z; x[r][NT / 4 - 1] = u.w;
      } else {
        const uint2 u = *reinterpret_cast<const uint2*>(vt + KdTile<D>::val(row, g >> 1) + 8 * (g & 1));
        x[r][0] = u.x; x[r][1] = u.y;
      }
    }
#pragma unroll
    for (int w = 0; w < NT / 4; w++) {
      const uint32_t a0 = __byte_perm(x[0][w], x[1][w], 0x5140), a1 = __byte_perm(x[0][w], x[1][w], 0x7362);
      const uint32_t c0 = __byte_perm(x[2][w], x[3][w], 0x5140), c1 = __byte_perm(x[2][w], x[3][w], 0x7362);
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const uint32_t b0 = kv8_half2((e < 2 ? a0 : a1) >> (16 * (e & 1))), b1 = kv8_half2((e < 2 ? c0 : c1) >> (16 * (e & 1)));
        kd_mma(o[4 * w + e], ph, b0, b1);
        if (TWO) kd_mma(o[4 * w + e], pl, b0, b1);
      }
    }
    __syncwarp();                              // every lane has read the stage that the next fetch fills
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");

  // ---- the four warps' results joined
#pragma unroll
  for (int h = 0; h < 2; h++) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    if (t == 0) { s_m[warp][g + 8 * h] = m[h]; s_l[warp][g + 8 * h] = l[h]; }
  }
  __syncthreads();                             // the rings are free as well
  float* so = reinterpret_cast<float*>(kd_smem);   // [warps][rows][kPitch]
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const int r = g + 8 * h;
    float M = s_m[0][r];
#pragma unroll
    for (int w = 1; w < kKdWarps; w++) M = fmaxf(M, s_m[w][r]);
    const float f = m[h] == -INFINITY ? 0.f : kd_exp2(m[h] - M);
    float* dst = so + (warp * kKdRows + r) * kPitch;
    // columns 2 t and 2 t + 1 of tile k are dims (2 t) D / 8 + k and (2 t + 1) D / 8 + k
#pragma unroll
    for (int e = 0; e < 2; e++)
#pragma unroll
      for (int k = 0; k < NT; k += 4)
        *reinterpret_cast<float4*>(dst + (2 * t + e) * (D / 8) + k) =
            make_float4(o[k][2 * h + e] * f, o[k + 1][2 * h + e] * f, o[k + 2][2 * h + e] * f, o[k + 3][2 * h + e] * f);
  }
  __syncthreads();
  const bool last = p.splits == 1;
  for (int c = tid; c < kKdRows * (D / 8); c += kKdWarps * 32) {
    const int r = c / (D / 8), d = c % (D / 8) * 8, row = m0 + r;
    if (row >= R) continue;
    float M = s_m[0][r];
#pragma unroll
    for (int w = 1; w < kKdWarps; w++) M = fmaxf(M, s_m[w][r]);
    float sum = 0.f, v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kKdWarps; w++) {
      sum += s_m[w][r] == -INFINITY ? 0.f : s_l[w][r] * kd_exp2(s_m[w][r] - M);
      const float* src = so + (w * kKdRows + r) * kPitch + d;
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] += src[j];
    }
    const int tok = sq.row + row / p.G, head = kvh * p.G + row % p.G;
    if (last) {
      if (p.sinks) sum += kd_exp2(p.sinks[head] * kLog2e - (M == -INFINITY ? 0.f : M));
      const float inv = sum > 0.f ? 1.f / sum : sum != sum ? sum : 0.f;
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] *= inv;
      Elems<T>::store(static_cast<T*>(p.out) + tok * p.out_stride + (int64_t)head * D + d, p.out_vec, v);
    } else {
      const size_t at = ((size_t)blockIdx.x * p.b.n_tokens + tok) * p.heads + head;
      Elems<float>::store(p.part + at * D + d, true, v);
      if (d == 0) *reinterpret_cast<float2*>(kv8_part_ml(p, D) + 2 * at) = make_float2(M, sum);
    }
  }
}

// The splits of one row joined, in their order; one block per (token, query head), a warp takes every fourth split.
template <class T, int D>
__global__ void __launch_bounds__(128) kv8_attn_join_kernel(const Kv8AttnParams p) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ float s_m[4], s_l[4];
  __shared__ __align__(16) float s_o[4][D];
  constexpr int V = D / 32;
  const int head = blockIdx.y, tok = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int s = kv8_find(p.b.n_seq, tok, [&](int i) { return __ldg(p.b.seq_start + i); });
  const Kv8Seq sq = kv8_seq(p.b, s, p.status);
  const int i = tok - sq.row;
  if (i < 0 || i >= sq.n) return;
  const int row = i * p.G + head % p.G, m0 = row / p.tile * p.tile, m1 = min(m0 + p.tile, sq.n * p.G);
  const Kv8Range kr = kv8_range(sq, m0, m1, p.G, p.window, kKdStep);
  const int n = (kr.hi - kr.lo + p.chunk - 1) / p.chunk;
  const size_t stride = (size_t)p.b.n_tokens * p.heads, at = (size_t)tok * p.heads + head;
  const float2* ml = reinterpret_cast<const float2*>(kv8_part_ml(p, D)) + at;
  const float* po = p.part + at * D + lane * V;
  float m = -INFINITY, l = 0.f, o[V];
#pragma unroll
  for (int j = 0; j < V; j++) o[j] = 0.f;
#pragma unroll 4
  for (int x = warp; x < n; x += 4) {
    const float2 a = __ldcg(ml + x * stride);
    float v[V];
#pragma unroll
    for (int j = 0; j < V; j += 2) {
      const float2 u = __ldcg(reinterpret_cast<const float2*>(po + x * stride * D + j));
      v[j] = u.x; v[j + 1] = u.y;
    }
    const float mn = fmaxf(m, a.x), f = m == -INFINITY ? 0.f : kd_exp2(m - mn), e = a.x == -INFINITY ? 0.f : kd_exp2(a.x - mn);
    m = mn;
    l = l * f + a.y * e;
#pragma unroll
    for (int j = 0; j < V; j++) o[j] = o[j] * f + v[j] * e;
  }
  if (lane == 0) { s_m[warp] = m; s_l[warp] = l; }
#pragma unroll
  for (int j = 0; j < V; j += 2) *reinterpret_cast<float2*>(&s_o[warp][lane * V + j]) = make_float2(o[j], o[j + 1]);
  __syncthreads();
  if (threadIdx.x >= D / 8) return;
  const int d = threadIdx.x * 8;
  const float M = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
  float sum = 0.f, v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int w = 0; w < 4; w++) {
    const float f = s_m[w] == -INFINITY ? 0.f : kd_exp2(s_m[w] - M);
    sum += s_l[w] * f;
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] += s_o[w][d + j] * f;
  }
  if (p.sinks) sum += kd_exp2(p.sinks[head] * kLog2e - (M == -INFINITY ? 0.f : M));
  const float inv = sum > 0.f ? 1.f / sum : sum != sum ? sum : 0.f;
#pragma unroll
  for (int j = 0; j < 8; j++) v[j] *= inv;
  Elems<T>::store(static_cast<T*>(p.out) + tok * p.out_stride + (int64_t)head * D + d, p.out_vec, v);
}

// ---------------------------------------------------------------- host side
struct Kv8Plan { int tiles, chunk, splits, most; };      // most: splits at most, for any window
static Kv8Plan kv8_plan(const Kv8Batch& b, int kv_heads, int heads, int window, int sms) {
  const int G = heads / kv_heads;
  Kv8Plan pl;
  pl.tiles = (int)(((int64_t)b.max_new * G + kKdRows - 1) / kKdRows);
  const int64_t units = (int64_t)pl.tiles * kv_heads * b.n_seq;
  // three blocks an SM; several sequences, whose lengths differ, in three waves
  const int64_t want = (int64_t)3 * sms * (b.n_seq > 1 ? 3 : 1);
  const Kv8Split sp = kv8_split(kv8_span(b.max_len, kKdRows, G, window, kKdStep), units, want, 128);
  pl.chunk = sp.chunk; pl.splits = sp.splits;
  pl.most = kv8_most_splits(b.max_len, units, want, 128);
  return pl;
}
static int kv8_sms(int* sms) {
  int dev = 0;
  MSB_CUDA(cudaGetDevice(&dev));
  MSB_CUDA(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev));
  return kOk;
}
static int kv8_heads_check(const msb_kv8_cache* c, int heads, const char* what) {
  if (heads <= 0 || heads > 65535 || heads % c->kv_heads) return fail(kErrArg, "%s: %d query heads over %d key heads", what, heads, c->kv_heads);
  return kOk;
}
static size_t kv8_part_bytes(const Kv8Batch& b, int heads, int D, int splits) {
  return splits > 1 ? sizeof(float) * (size_t)splits * b.n_tokens * heads * (D + 2) : 0;
}
size_t kv8_attn_scratch_bytes(const msb_kv8_cache* c, const msb_kv8_batch* b, int heads) {
  Kv8Cache cc; Kv8Batch bb;
  int sms;
  if (kv8_check(c, b, "kv8_attn_scratch_bytes", &cc, &bb) || kv8_heads_check(c, heads, "kv8_attn_scratch_bytes") || kv8_sms(&sms)) return 0;
  return 16 + kv8_part_bytes(bb, heads, c->head_dim, kv8_plan(bb, cc.heads, heads, 0, sms).most);
}

template <class T, int D>
static int launch_attn(Kv8AttnParams& p, const Kv8Plan& pl, cudaStream_t st, int dev) {
  auto kern = kv8_attn_few_kernel<T, D>;
  const size_t smem = std::max<size_t>((size_t)kKdWarps * kKdStages * 2 * KdTile<D>::kBytes, sizeof(float) * kKdWarps * kKdRows * (D + 4));
  static bool done[64] = {};
  if (!done[dev & 63]) {
    MSB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
    done[dev & 63] = true;
  }
  MSB_CUDA(launch_pdl(kern, dim3(pl.splits, p.c.heads * pl.tiles, p.b.n_seq), dim3(kKdWarps * 32), smem, st, p));
  MSB_LAUNCH_CHECK("kv8_attn");
  if (pl.splits > 1) {
    MSB_CUDA(launch_pdl(kv8_attn_join_kernel<T, D>, dim3(p.b.n_tokens, p.heads), dim3(128), 0, st, p));
    MSB_LAUNCH_CHECK("kv8_attn_join");
  }
  return kOk;
}

int kv8_attn(const msb_kv8_cache* c, const msb_kv8_batch* b, int elem_type, const void* q, int64_t q_stride, int heads, float scale,
             int window, const float* sinks, void* out, int64_t out_stride, void* scratch, size_t scratch_bytes, cudaStream_t st) {
  const char* what = "kv8_attn";
  Kv8AttnParams p{};
  int rc = kv8_check(c, b, what, &p.c, &p.b);
  if (rc || (rc = kv8_heads_check(c, heads, what))) return rc;
  bool qv, ov;
  if ((rc = kv8_rows_check(q, q_stride, heads, c->head_dim, elem_type, what, &qv))) return rc;
  if ((rc = kv8_rows_check(out, out_stride, heads, c->head_dim, elem_type, what, &ov))) return rc;
  if (window < 0) return fail(kErrArg, "%s: window %d", what, window);
  if (!(scale == scale) || scale - scale != 0.f) return fail(kErrArg, "%s: scale is not a number", what);
  int dev, sms;
  MSB_CUDA(cudaGetDevice(&dev));
  if ((rc = kv8_sms(&sms))) return rc;
  const Kv8Plan pl = kv8_plan(p.b, p.c.heads, heads, window, sms);
  if ((int64_t)p.c.heads * pl.tiles > 65535) return fail(kErrLimit, "%s: too many rows", what);
  const size_t need = kv8_part_bytes(p.b, heads, c->head_dim, pl.splits);
  if (need && (!scratch || scratch_bytes < need)) return fail(kErrScratch, "%s: scratch too small (%zu < %zu)", what, scratch_bytes, need);
  if (need && (reinterpret_cast<uintptr_t>(scratch) & 15)) return fail(kErrArg, "%s: scratch must be 16-byte aligned", what);
  Tables tb;
  if ((rc = get_tables(&tb))) return rc;
  p.q = q; p.out = out; p.q_stride = q_stride; p.out_stride = out_stride; p.sinks = sinks; p.part = static_cast<float*>(scratch);
  p.scale = scale; p.heads = heads; p.G = heads / p.c.heads; p.window = window; p.chunk = pl.chunk; p.splits = pl.splits; p.tile = kKdRows;
  p.q_vec = qv; p.out_vec = ov; p.status = tb.status;
#define KV8_GO(T) return c->head_dim == 64 ? launch_attn<T, 64>(p, pl, st, dev) : launch_attn<T, 128>(p, pl, st, dev)
  if (elem_type == F32) KV8_GO(float);
  if (elem_type == F16) KV8_GO(__half);
  KV8_GO(__nv_bfloat16);
#undef KV8_GO
}

}  // namespace msb
