// Attention over the 8-bit cache (kv8_attn.cuh) for few query rows: single tokens and short drafts.
//
// Every code is read once and what bounds the kernel is that read.  A block of four warps takes 16 rows of one key head (mma.sync
// m16n8k16: a whole group of query heads, several tokens of a draft) over one range of keys; a warp takes every fourth step of 32 tokens.
// Steps are fetched by the warp itself, with cp.async into its own two buffers, so that the warps never wait for one another before the end.
//   scores   the contraction may run over the dims in any order: a lane takes 16 neighbouring bytes of "its" token as eight pairs and
//            the query's registers are laid out alike; a pair of codes is one conversion to two halves (exact)
//   output   the tokens are contracted: bytes of two neighbouring tokens are interleaved and converted; lane g holds dims [g D / 8, (g + 1) D / 8)
//   weights  the reference of the exponents moves only when a weight would pass 2^15 (a half ends at 2^16), and then so that it becomes 2^11: the
//            sums are rescaled a few times, not at every new maximum.  A half holds nothing below 2^-25: what a warp's N keys lose beside the
//            largest of them is N 2^-36 at most
// The queries are scaled by a power of two to at most 2 in a row and used as halves; F32 ones, and their weights, as two halves each.
#include <algorithm>
#include "kv8_attn.cuh"

namespace msb {

constexpr int kKdCluster = 8;      // blocks of a cluster at most
constexpr float kKdTop = 15.f, kKdFirst = 11.f;      // exponents of a weight: above which the reference moves, and then
constexpr int kKdFold = 16;         // steps of a warp after which F32 rows' sums begin anew
constexpr int kKdWarps = 4, kKdStages = 2, kKdStep = kKv8FewStep, kKdRows = kKv8FewRows;

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
  // where 16-byte chunk c of row r lies.  D 128: the keys' reads (rows r, r + 1; chunks t, t + 4) and the values' (rows 2 t, chunks g) are
  // free of bank conflicts with these; D 64: rows 4..7 and 12..15 change places in pairs as well
  static __device__ __forceinline__ uint32_t key(int r, int c) { return D == 128 ? r * 128 + ((c ^ ((r & 1) << 2)) << 4) : r * 64 + (c << 4); }
  static __device__ __forceinline__ uint32_t val(int r, int c) {
    return D == 128 ? r * 128 + ((c ^ (r & 6)) << 4) : (r ^ ((r >> 2) & 1)) * 64 + ((c ^ (((r >> 1) & 1) << 1)) << 4);
  }
};

__device__ __forceinline__ void kd_cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t kd_of_block(const void* p, uint32_t rank) {      // the same shared variable of another block of the cluster
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ float kd_load_of(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 kd_load4_of(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

// Blocks of an SM: F32 rows of 128 dims need more registers than a third of an SM's threads have (64 ragged sequences: 150 us with two blocks,
// 211 with three and 270 bytes a thread in local memory).  Four of 64 dims gain nothing (200K tokens, bf16: 44 us with three).
constexpr int kd_blocks(bool f32, int dim) { return f32 && dim == 128 ? 2 : 3; }
// CLUSTER: the parts of a row are the blocks of a cluster, which join them through one another's shared memory
template <class T, int D, bool CLUSTER>
__global__ void __launch_bounds__(kKdWarps * 32, kd_blocks(sizeof(T) == 4, D)) kv8_attn_few_kernel(const Kv8AttnParams p) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr bool TWO = sizeof(T) == 4;
  constexpr int KS = D / 16, NT = D / 8, CH = D / 64;      // k-steps, output tiles, 16-byte chunks of a key row per lane
  constexpr int kHalf = 16 * D, kStage = 4 * kHalf, kWarpBytes = kKdStages * kStage, kPitch = D + 4;     // keys of 32 tokens, their values
  extern __shared__ __align__(16) uint8_t kd_smem[];
  __shared__ float s_m[kKdWarps][kKdRows], s_l[kKdWarps][kKdRows], s_bm[kKdRows], s_bl[kKdRows];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int tiles = gridDim.y / p.c.heads, kvh = blockIdx.y / tiles, m0 = (blockIdx.y % tiles) * kKdRows;
  // without a window the keys of this part are known before the sequence is: its first blocks' ids are asked for at the same time
  const int* table = p.b.table + (size_t)blockIdx.z * p.b.table_stride;
  const int early = (blockIdx.x * p.chunk + kKdStep * (warp + kKdWarps * (lane >> 1)) + 16 * (lane & 1)) >> p.c.shift;
  const int early_id = early < p.b.table_stride ? __ldg(table + early) : -1;
  const Kv8Seq sq = kv8_seq(p.b, blockIdx.z, p.status);
  const int R = sq.n * p.G;
  if (m0 >= R) return;
  const int m1 = min(m0 + kKdRows, R);
  const Kv8Range kr = kv8_range(sq, m0, m1, p.G, p.window, kKdStep);
  const int k0 = kr.lo + blockIdx.x * p.chunk, k1 = min(kr.hi, k0 + p.chunk);
  if (!CLUSTER && k0 >= k1) return;
  const int steps = k1 > k0 ? (k1 - k0 + kKdStep - 1) / kKdStep : 0;
  const int mine = steps > warp ? (steps - warp + kKdWarps - 1) / kKdWarps : 0;

  // ---- block ids and scales of the warp's next 16 steps, half a step (16 tokens: one block) per lane; ve = -inf: no such block
  int ids = -1;
  float ksc = 0.f, vex = -INFINITY;
  auto look_up = [&](int i) {
    const int key = k0 + kKdStep * (warp + kKdWarps * (i + (lane >> 1))) + 16 * (lane & 1);
    ids = -1; ksc = 0.f; vex = -INFINITY;
    if (key < k1 && key + 16 > kr.first) {
      ids = i == 0 && kr.lo == 0 ? early_id : __ldg(table + (key >> p.c.shift));
      if (ids < 0 || ids >= p.c.n_blocks) { ids = -1; atomicCAS(p.status, 0, kDevBadBatch); }
      else {
        ksc = __ldg(p.c.ks + (size_t)ids * p.c.heads + kvh);
        vex = (float)kv8_exp(__ldg(p.c.vs + (size_t)ids * p.c.heads + kvh));
      }
    }
  };
  // this lane's part of a copy: 16 bytes of rows r0, r0 + 512 / D, ...
  const int r0 = lane / (D / 16), c0 = lane % (D / 16);
  const uint32_t ring = smem_u32(kd_smem) + warp * kWarpBytes;
  const uint32_t kd = ring + KdTile<D>::key(r0, c0);
  const uint32_t vd[2] = {ring + 2 * kHalf + KdTile<D>::val(r0, c0), ring + 2 * kHalf + KdTile<D>::val(r0 + 512 / D, c0) - 512};
  const uint8_t *ksrc = p.c.k + 16 * lane, *vsrc = p.c.v + 16 * lane;
  auto fetch = [&](int i) {                   // step i of the warp; its lane's ids are loaded
    if (i < mine) {
      const int base = k0 + kKdStep * (warp + kKdWarps * i);
      const uint32_t st = (i & 1) * kStage;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int id = __shfl_sync(0xffffffffu, ids, (2 * i + h) & 31), key = base + 16 * h;
        const int rows = id >= 0 ? sq.len - key - r0 : 0;      // rows behind the last token hold anything: zeros for them
        const size_t off = ((((size_t)max(id, 0) * p.c.heads + kvh) << p.c.shift) + (key & ((1 << p.c.shift) - 1))) * D;
#pragma unroll
        for (int j = 0; j < D / 32; j++) {
          const bool there = rows > j * (512 / D);
          kd_copy16(kd + st + h * kHalf + 512 * j, ksrc + off + 512 * j, there);
          kd_copy16(vd[j & 1] + st + h * kHalf + 512 * j, vsrc + off + 512 * j, there);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  look_up(0);
  float ks_cur = ksc, ve_cur = vex;           // of the batch that is being computed (the fetches run ahead into the next one)
  fetch(0);

  // ---- queries: rows g and g + 8 of the tile, scaled to at most 2
  uint32_t qh[KS][4], ql[TWO ? KS : 1][4];
  float qs[2];
  int qpos[2];
#pragma unroll
  for (int h = 0; h < 2; h++) {
    const int r = m0 + g + 8 * h, tok = min(r, R - 1) / p.G, head = kvh * p.G + min(r, R - 1) % p.G;
    const T* src = static_cast<const T*>(p.q) + (sq.row + tok) * p.q_stride + (int64_t)head * D;
    qpos[h] = sq.len - sq.n + tok;
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
    const int e = min(max((int)(__float_as_uint(top) >> 23) - 127, -126), 120);
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
  // keys that every row of the tile sees: no comparisons for steps inside them
  const int all_hi = min(k1, sq.len - sq.n + m0 / p.G + 1), all_lo = p.window ? sq.len - sq.n + (m1 - 1) / p.G - p.window + 1 : 0;

  float o[NT][4];
#pragma unroll
  for (int i = 0; i < NT; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  const uint8_t* own = kd_smem + warp * kWarpBytes;
  float4* sums = reinterpret_cast<float4*>(kd_smem + kKdWarps * kWarpBytes) + warp * NT * 32 + lane;      // F32: this lane's share of what O held
  const uint8_t* kl = own + KdTile<D>::key(g, t);
  const uint8_t* vl[2] = {own + 2 * kHalf + KdTile<D>::val(2 * t, D == 128 ? g : g >> 1) + (D == 128 ? 0 : 8 * (g & 1)),
                          own + 2 * kHalf + KdTile<D>::val(2 * t + 1, D == 128 ? g : g >> 1) + (D == 128 ? 0 : 8 * (g & 1))};
  const int flip = (g & 1) ? -64 : 64;        // a key row's other chunk (D 128)

  for (int i = 0; i < mine; i++) {
    if (i + 1 < mine && ((i + 1) & 15) == 0) look_up(i + 1);
    fetch(i + 1);
    if (i && (i & 15) == 0) { ks_cur = ksc; ve_cur = vex; }
    if (TWO && i && i % kKdFold == 0) {       // the tensor core cuts off what its sums do not hold: they begin anew, and what they held is added up
#pragma unroll
      for (int k = 0; k < NT; k++) {
        float4 a = make_float4(o[k][0], o[k][1], o[k][2], o[k][3]);
        if (i > kKdFold) { const float4 b = sums[32 * k]; a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w; }
        sums[32 * k] = a;
        o[k][0] = o[k][1] = o[k][2] = o[k][3] = 0.f;
      }
    }
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncwarp();
    const uint32_t st = (i & 1) * kStage;
    const int base = k0 + kKdStep * (warp + kKdWarps * i);
    float ks[2], ve[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
      ks[h] = __shfl_sync(0xffffffffu, ks_cur, (2 * i + h) & 31);
      ve[h] = __shfl_sync(0xffffffffu, ve_cur, (2 * i + h) & 31);
    }
    // ---- scores of 32 tokens
    float s[4][4];
#pragma unroll
    for (int nt = 0; nt < 4; nt++) s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
#pragma unroll
    for (int j = 0; j < CH; j++) {
      uint32_t w[4][4];
#pragma unroll
      for (int nt = 0; nt < 4; nt++) {
        const uint4 u = *reinterpret_cast<const uint4*>(kl + st + nt * 8 * D + (j ? flip : 0));
        w[nt][0] = u.x; w[nt][1] = u.y; w[nt][2] = u.z; w[nt][3] = u.w;
      }
#pragma unroll
      for (int x = 0; x < 4; x++)
#pragma unroll
        for (int nt = 0; nt < 4; nt++) {
          const uint32_t b0 = kv8_half2(w[nt][x]), b1 = kv8_half2(w[nt][x] >> 16);
          kd_mma(s[nt], qh[4 * j + x], b0, b1);
          if (TWO) kd_mma(s[nt], ql[4 * j + x], b0, b1);
        }
    }
    // ---- weights: rows (r >> 1), tokens 8 nt + 2 t + (r & 1)
#pragma unroll
    for (int nt = 0; nt < 4; nt++)
#pragma unroll
      for (int r = 0; r < 4; r++) s[nt][r] = fmaf(s[nt][r], qs[r >> 1] * ks[nt >> 1], ve[nt >> 1]);
    if (base + kKdStep > all_hi || base < all_lo) {
#pragma unroll
      for (int nt = 0; nt < 4; nt++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const int key = base + 8 * nt + 2 * t + (r & 1), pos = qpos[r >> 1];
          if (key >= k1 || key > pos || (p.window && key <= pos - p.window)) s[nt][r] = -INFINITY;
        }
    }
    float top[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
      top[h] = fmaxf(fmaxf(fmaxf(s[0][2 * h], s[0][2 * h + 1]), fmaxf(s[1][2 * h], s[1][2 * h + 1])),
                     fmaxf(fmaxf(s[2][2 * h], s[2][2 * h + 1]), fmaxf(s[3][2 * h], s[3][2 * h + 1])));
      top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
      top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
    }
    if (__any_sync(0xffffffffu, top[0] - m[0] > kKdTop || top[1] - m[1] > kKdTop)) {      // (-infinity twice: no)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const float n = top[h] - m[h] > kKdTop ? top[h] - (fabsf(top[h]) < 1e6f ? kKdFirst : 0.f) : m[h], f = n == -INFINITY ? 1.f : kd_exp2(m[h] - n);
        m[h] = n; l[h] *= f;
#pragma unroll
        for (int k = 0; k < NT; k++) { o[k][2 * h] *= f; o[k][2 * h + 1] *= f; }
        if (TWO && i >= kKdFold)
#pragma unroll 1
          for (int k = 0; k < NT; k++) {
            float2* b = reinterpret_cast<float2*>(sums + 32 * k) + h;
            *b = make_float2(b->x * f, b->y * f);
          }
      }
    }
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const float mm = m[h] == -INFINITY ? 0.f : m[h];
#pragma unroll
      for (int x = 0; x < 2; x++) {           // halves of the step: a block and its value scale each
        float sum = 0.f;
#pragma unroll
        for (int y = 0; y < 4; y++) {
          float& v = s[2 * x + (y >> 1)][2 * h + (y & 1)];
          v = kd_exp2(v - mm);
          sum += v;
        }
        l[h] = fmaf(sum, ve[x] == -INFINITY ? 0.f : kv8_pow2(-(int)ve[x]), l[h]);
      }
    }
    // ---- output
#pragma unroll
    for (int h = 0; h < 2; h++) {
      uint32_t ph[4], pl[4], x[4][NT / 4];
      kd_split<TWO>(s[2 * h][0], s[2 * h][1], ph[0], pl[0]);
      kd_split<TWO>(s[2 * h][2], s[2 * h][3], ph[1], pl[1]);
      kd_split<TWO>(s[2 * h + 1][0], s[2 * h + 1][1], ph[2], pl[2]);
      kd_split<TWO>(s[2 * h + 1][2], s[2 * h + 1][3], ph[3], pl[3]);
#pragma unroll
      for (int r = 0; r < 4; r++) {           // rows 2 t, 2 t + 1, 2 t + 8, 2 t + 9
        const uint8_t* src = vl[r & 1] + st + h * kHalf + (r >> 1) * 8 * D;
        if (D == 128) {
          const uint4 u = *reinterpret_cast<const uint4*>(src);
          x[r][0] = u.x; x[r][1] = u.y; x[r][NT / 4 - 2] = u.z; x[r][NT / 4 - 1] = u.w;
        } else {
          const uint2 u = *reinterpret_cast<const uint2*>(src);
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
    }
    __syncwarp();                              // every lane has read the buffer that the next fetch fills
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  if (TWO && mine > kKdFold)
#pragma unroll
    for (int k = 0; k < NT; k++) {
      const float4 b = sums[32 * k];
      o[k][0] += b.x; o[k][1] += b.y; o[k][2] += b.z; o[k][3] += b.w;
    }

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
    if (CLUSTER) {                             // in place: nobody else reads these eight
      Elems<float>::store(so + r * kPitch + d, true, v);
      if (d == 0) { s_bm[r] = M; s_bl[r] = sum; }
    } else if (last) {
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
  if (CLUSTER) {
    kd_cluster_sync();
    const int n = gridDim.x;                   // blocks of the cluster: each writes a share of the rows
    for (int c = tid + kKdWarps * 32 * blockIdx.x; c < (m1 - m0) * (D / 8); c += kKdWarps * 32 * n) {
      const int r = c / (D / 8), d = c % (D / 8) * 8, row = m0 + r, tok = sq.row + row / p.G, head = kvh * p.G + row % p.G;
      float M = -INFINITY, sum = 0.f, v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, m[kKdCluster], l[kKdCluster];
#pragma unroll
      for (int b = 0; b < kKdCluster; b++) {   // all of them requested before the first is used
        m[b] = b < n ? kd_load_of(kd_of_block(&s_bm[r], b)) : -INFINITY;
        l[b] = b < n ? kd_load_of(kd_of_block(&s_bl[r], b)) : 0.f;
      }
#pragma unroll
      for (int b = 0; b < kKdCluster; b++) M = fmaxf(M, m[b]);
#pragma unroll
      for (int h = 0; h < kKdCluster; h += 4) {
        float4 x[4], y[4];
#pragma unroll
        for (int b = 0; b < 4; b++) {
          const uint32_t src = kd_of_block(so + r * kPitch + d, min(h + b, n - 1));
          x[b] = kd_load4_of(src); y[b] = kd_load4_of(src + 16);
        }
#pragma unroll
        for (int b = 0; b < 4; b++) {
          const float f = m[h + b] == -INFINITY ? 0.f : kd_exp2(m[h + b] - M);      // (and of a block that is not there)
          sum += l[h + b] * f;
          v[0] += x[b].x * f; v[1] += x[b].y * f; v[2] += x[b].z * f; v[3] += x[b].w * f;
          v[4] += y[b].x * f; v[5] += y[b].y * f; v[6] += y[b].z * f; v[7] += y[b].w * f;
        }
      }
      if (p.sinks) sum += kd_exp2(p.sinks[head] * kLog2e - (M == -INFINITY ? 0.f : M));
      const float inv = sum > 0.f ? 1.f / sum : sum != sum ? sum : 0.f;
#pragma unroll
      for (int j = 0; j < 8; j++) v[j] *= inv;
      Elems<T>::store(static_cast<T*>(p.out) + tok * p.out_stride + (int64_t)head * D + d, p.out_vec, v);
    }
    kd_cluster_sync();                         // no block leaves while another reads its memory
  }
}

// The splits of one row joined, in their order: WARPS warps a (token, query head), each every WARPS-th split.
template <class T, int D, int WARPS>
__global__ void __launch_bounds__(128) kv8_attn_join_kernel(const Kv8AttnParams p) {
  pdl_launch_dependents();
  pdl_wait();
  constexpr int V = D / 32, kRows = 4 / WARPS;
  __shared__ float s_m[4], s_l[4];
  __shared__ __align__(16) float s_o[4][D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, part = warp % WARPS;
  const int64_t at = (int64_t)blockIdx.x * kRows + warp / WARPS;        // row of the rows' products: token * heads + head
  const int tok = (int)(at / p.heads), head = (int)(at - (int64_t)tok * p.heads);
  int n = 0;
  if (tok < p.b.n_tokens) {
    Kv8Seq sq;
    const int s = kv8_owner(p.b.n_seq, tok, [&](int i) { return kv8_seq(p.b, i, p.status); }, [&](int i) { return __ldg(p.b.seq_start + i); },
                            [](auto f) { return __ballot_sync(0xffffffffu, f(threadIdx.x & 31)); }, sq);
    const int i = tok - sq.row;
    if (s >= 0) {
      const int row = i * p.G + head % p.G, m0 = row / p.tile * p.tile, m1 = min(m0 + p.tile, sq.n * p.G);
      const Kv8Range kr = kv8_range(sq, m0, m1, p.G, p.window, p.step);
      n = (kr.hi - kr.lo + p.chunk - 1) / p.chunk;
    }
  }
  const size_t stride = (size_t)p.b.n_tokens * p.heads;
  const float2* ml = reinterpret_cast<const float2*>(kv8_part_ml(p, D)) + at;
  const float* po = p.part + at * D + lane * V;
  float m = -INFINITY, l = 0.f, o[V];
#pragma unroll
  for (int j = 0; j < V; j++) o[j] = 0.f;
#pragma unroll 4
  for (int x = part; x < n; x += WARPS) {
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
  if (WARPS == 1) __syncwarp();
  else __syncthreads();
  if (n == 0 || part || lane >= D / 8) return;
  const int d = lane * 8;
  float M = s_m[warp];
#pragma unroll
  for (int w = 1; w < WARPS; w++) M = fmaxf(M, s_m[warp + w]);
  float sum = 0.f, v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int w = 0; w < WARPS; w++) {
    const float f = s_m[warp + w] == -INFINITY ? 0.f : kd_exp2(s_m[warp + w] - M);
    sum += s_l[warp + w] * f;
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] += s_o[warp + w][d + j] * f;
  }
  if (p.sinks) sum += kd_exp2(p.sinks[head] * kLog2e - (M == -INFINITY ? 0.f : M));
  const float inv = sum > 0.f ? 1.f / sum : sum != sum ? sum : 0.f;
#pragma unroll
  for (int j = 0; j < 8; j++) v[j] *= inv;
  Elems<T>::store(static_cast<T*>(p.out) + tok * p.out_stride + (int64_t)head * D + d, p.out_vec, v);
}

// ---------------------------------------------------------------- host side
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
// the parts with their references and sums, or, for one part whose sums are begun anew (kv8_attn_many), what they held
static size_t kv8_part_bytes(const Kv8Batch& b, int heads, int D, int splits, bool folds) {
  return splits > 1 ? sizeof(float) * (size_t)splits * b.n_tokens * heads * (D + 2) : folds ? sizeof(float) * (size_t)b.n_tokens * heads * D : 0;
}
size_t kv8_attn_scratch_bytes(const msb_kv8_cache* c, const msb_kv8_batch* b, int heads) {      // for rows of any type
  Kv8Cache cc; Kv8Batch bb;
  int sms;
  if (kv8_check(c, b, "kv8_attn_scratch_bytes", &cc, &bb) || kv8_heads_check(c, heads, "kv8_attn_scratch_bytes") || kv8_sms(&sms)) return 0;
  // (a window may change which kernel runs, and a split that is none needs no room)
  int most = 1;
  for (int f32 = 0; f32 < 2; f32++) {
    const Kv8Most m = kv8_most(bb.n_seq, bb.max_new, bb.max_len, cc.heads, heads, f32, sms);
    most = std::max(most, std::max(m.few, m.many));
  }
  return 16 + kv8_part_bytes(bb, heads, c->head_dim, most, bb.max_len > kKv8Fold);
}

template <class T, int D>
static int launch_attn(const Kv8AttnParams& p, const Kv8Plan& pl, int elem_type, cudaStream_t st, int dev, int sms) {
  if (pl.many) {
    const int rc = kv8_attn_many(p, pl.tiles, elem_type, D, st, dev);
    if (rc) return rc;
  } else {
    const size_t ring = (size_t)kKdWarps * kKdStages * 2 * kKdStep * D, sums = sizeof(T) == 4 ? sizeof(float) * kKdWarps * kKdRows * D : 0;
    const size_t smem = std::max(ring + sums, sizeof(float) * kKdWarps * kKdRows * (D + 4));
    static bool done[64] = {};
    if (!done[dev & 63]) {
      MSB_CUDA(cudaFuncSetAttribute(kv8_attn_few_kernel<T, D, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
      MSB_CUDA(cudaFuncSetAttribute(kv8_attn_few_kernel<T, D, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
      done[dev & 63] = true;
    }
    const dim3 grid(pl.splits, p.c.heads * pl.tiles, p.b.n_seq);
    // few parts of few rows: one launch, the parts a cluster (a token of 64 heads over 8 behind 998: F32: 11.2 us with a second launch, 8.1).  Not once the blocks do
    // not all run at once: those of short sequences would wait for the long ones of their cluster
    if (pl.splits > 1 && pl.splits <= kKdCluster && (int64_t)grid.x * grid.y * grid.z <= 2 * sms) {
      MSB_CUDA(launch_clusters(kv8_attn_few_kernel<T, D, true>, grid, dim3(kKdWarps * 32), pl.splits, smem, st, p));
      MSB_LAUNCH_CHECK("kv8_attn");
      return kOk;
    }
    MSB_CUDA(launch_pdl(kv8_attn_few_kernel<T, D, false>, grid, dim3(kKdWarps * 32), smem, st, p));
    MSB_LAUNCH_CHECK("kv8_attn");
  }
  if (pl.splits > 1) {
    // a warp a row for few parts or many rows, four where a row's parts would be a long chain
    const int64_t rows = (int64_t)p.b.n_tokens * p.heads;
    const bool alone = pl.splits <= 8 || rows >= 32768;
    MSB_CUDA(launch_pdl(alone ? kv8_attn_join_kernel<T, D, 1> : kv8_attn_join_kernel<T, D, 4>, dim3((unsigned)(alone ? (rows + 3) / 4 : rows)),
                        dim3(128), 0, st, p));
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
  if (reinterpret_cast<uintptr_t>(sinks) & 3) return fail(kErrArg, "%s: sinks are not aligned to F32", what);
  if (window < 0) return fail(kErrArg, "%s: window %d", what, window);
  if (!(scale == scale) || scale - scale != 0.f) return fail(kErrArg, "%s: scale is not a number", what);
  int dev, sms;
  MSB_CUDA(cudaGetDevice(&dev));
  if ((rc = kv8_sms(&sms))) return rc;
  const Kv8Plan pl = kv8_plan(p.b.n_seq, p.b.max_new, p.b.max_len, p.c.heads, heads, c->head_dim, elem_type == F32, window, sms);
  if (pl.many && pl.tiles > 65535) return fail(kErrLimit, "%s: too many rows", what);
  if ((int64_t)p.b.n_tokens * heads > 0x7fffffff) return fail(kErrLimit, "%s: too many rows", what);
  const size_t need = kv8_part_bytes(p.b, heads, c->head_dim, pl.splits, pl.many && elem_type != F32 && pl.chunk > kKv8Fold);
  if (need && (!scratch || scratch_bytes < need)) return fail(kErrScratch, "%s: scratch too small (%zu < %zu)", what, scratch_bytes, need);
  if (need && (reinterpret_cast<uintptr_t>(scratch) & 15)) return fail(kErrArg, "%s: scratch must be 16-byte aligned", what);
  Tables tb;
  if ((rc = get_tables(&tb))) return rc;
  p.q = q; p.out = out; p.q_stride = q_stride; p.out_stride = out_stride; p.sinks = sinks; p.part = static_cast<float*>(scratch);
  p.scale = scale; p.heads = heads; p.G = heads / p.c.heads; p.window = window; p.chunk = pl.chunk; p.splits = pl.splits;
  p.tile = pl.rows; p.step = pl.step;
  p.q_vec = qv; p.out_vec = ov; p.status = tb.status;
#define KV8_GO(T) return c->head_dim == 64 ? launch_attn<T, 64>(p, pl, elem_type, st, dev, sms) : launch_attn<T, 128>(p, pl, elem_type, st, dev, sms)
  if (elem_type == F32) KV8_GO(float);
  if (elem_type == F16) KV8_GO(__half);
  KV8_GO(__nv_bfloat16);
#undef KV8_GO
}

}  // namespace msb
