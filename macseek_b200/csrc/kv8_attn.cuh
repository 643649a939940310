// Attention over the 8-bit cache: what the kernels for few and for many query rows, and the one that joins partial results, share.
//   row r of a (sequence, key head): token r / G of the sequence's new ones, query head r % G of the key head's group of G;
//   it sees the tokens j with pos - window < j <= pos, pos = kv_len - new + r / G (window 0: all up to pos)
//   l_j = scale q . k_j ;  out = sum_j exp(l_j - M) v_j / (sum_j exp(l_j - M) + exp(sink - M)), 0 where nothing is seen and no sink
// In base 2, with the value scale of token j's block (2^e_j) carried by the weight: w_j = 2^(l_j log2(e) + e_j - m), m the running
// maximum of that exponent, so that out = sum w_j code_j / sum w_j 2^-e_j and w_j <= 1 whatever the scales of the blocks are.
#pragma once
#include "kv8.cuh"

namespace msb {

constexpr float kLog2e = 1.4426950408889634f;

struct Kv8AttnParams {
  Kv8Cache c;
  Kv8Batch b;
  const void* q;
  void* out;
  int64_t q_stride, out_stride;
  const float* sinks;
  float* part;                 // [splits][n_tokens * heads][D], then [splits][n_tokens * heads] of (m, sum); one part: of its sums at most
  float scale;
  int heads, G, window;
  int chunk, splits, tile, step;   // keys of one split (a multiple of step), splits at most, rows of a tile, keys of a step
  int q_vec, out_vec;
  int* status;
};

// the kernel for many rows over `groups` blocks of rows
int kv8_attn_many(const Kv8AttnParams& p, int groups, int elem_type, int D, cudaStream_t st, int dev);

#ifdef __CUDACC__
__device__ __forceinline__ float* kv8_part_ml(const Kv8AttnParams& p, int D) {
  return p.part + (size_t)p.splits * p.b.n_tokens * p.heads * D;
}
#endif

}  // namespace msb
