// Index arithmetic of the 8-bit cache's kernels as plain C++, for the kernels and for tests on the host: which rows, blocks and keys a
// block of threads works on, for any contents of a batch's device arrays.  Nothing here gives an index outside what the arguments allow.
#pragma once
#include <cstdint>

#ifdef __CUDACC__
#define KV8_HD __host__ __device__ __forceinline__
#else
#define KV8_HD inline
#endif

namespace msb {

KV8_HD int kv8_min(int a, int b) { return a < b ? a : b; }
KV8_HD int kv8_max(int a, int b) { return a > b ? a : b; }

struct Kv8Seq { int row, n, len; };    // first row, new tokens, tokens with them

// A sequence from its entries in seq_start and kv_len; an empty one where they cannot be right.
KV8_HD bool kv8_seq_of(int r0, int r1, int len, int n_tokens, int max_new, int max_len, Kv8Seq& q) {
  const bool ok = r0 >= 0 && r1 >= r0 && r1 <= n_tokens && r1 - r0 <= max_new && len >= r1 - r0 && len <= max_len;
  q = ok ? Kv8Seq{r0, r1 - r0, len} : Kv8Seq{0, 0, 0};
  return ok;
}

// Work items of the kernels that go over the blocks which hold new tokens: n new tokens lie in at most (n >> shift) + 2 blocks, so
// sequence s owns the items from kv8_first_item on, and kv8_items are enough for any batch.
KV8_HD int kv8_first_item(int start, int s, int shift) { return (start >> shift) + 2 * s; }
inline int64_t kv8_items(int n_tokens, int n_seq, int shift) { return (int64_t)(n_tokens >> shift) + 2 * (int64_t)n_seq; }

// blocks that `n` new tokens lie in, at most
inline int kv8_touched(int n, int shift) { return (int)(((int64_t)n + (2 << shift) - 2) >> shift); }

// The j-th item of a sequence: its block's place in the table, first row, first token inside the block, tokens (0: nothing to do).
struct Kv8Item { int blk, row, at, n; };
KV8_HD Kv8Item kv8_item_of(const Kv8Seq& q, int j, int shift) {
  const int p0 = q.len - q.n, blk = (p0 >> shift) + j;
  if (j < 0 || q.n == 0 || blk > ((q.len - 1) >> shift)) return Kv8Item{0, 0, 0, 0};
  const int lo = kv8_max(p0, blk << shift), hi = kv8_min(q.len - (blk << shift), 1 << shift) + (blk << shift);
  return Kv8Item{blk, q.row + lo - p0, lo - (blk << shift), hi - lo};
}

// The last s with first(s) <= x, first(0) counted as no larger than x; first() rises (where it does not, some s of [0, n)).  Looked at
// by the 32 lanes of a warp at a time: ballot(f) is the mask of f(lane).
template <class First, class Ballot>
KV8_HD int kv8_search(int n, int x, First first, Ballot ballot) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32;
    const unsigned m = ballot([&](int lane) { return lane == 0 || (lane * (int64_t)step < hi - lo && first(lo + lane * step) <= x); });
    int c = 0;
    while (c < 32 && (m >> c & 1)) c++;
    lo += (c - 1) * step;
    hi = kv8_min(hi, lo + step);
  }
  return lo;
}

// Keys that rows [m0, m1) of a sequence look at (row r is token r / G of its new ones): [lo, hi), lo rounded down to `step`.
struct Kv8Range { int lo, hi; };
KV8_HD Kv8Range kv8_range(const Kv8Seq& s, int m0, int m1, int G, int window, int step) {
  const int p0 = s.len - s.n;
  Kv8Range r{0, p0 + (m1 - 1) / G + 1};
  if (window && p0 + m0 / G >= window) r.lo = (p0 + m0 / G - window + 1) / step * step;
  return r;
}
// most keys that a tile of `rows` rows looks at, for any sequence
inline int kv8_span(int max_len, int rows, int G, int window, int step) {
  const int64_t w = (int64_t)window + rows / G + 1 + step;
  return window && w < max_len ? (int)w : max_len;
}

// Split of the keys: `units` blocks of threads without one, about `want` blocks wanted; chunks of at least `least` keys, a multiple of `step`.
struct Kv8Split { int chunk, splits; };
inline Kv8Split kv8_split(int span, int64_t units, int64_t want, int least, int step = 64) {
  const int64_t n = want / (units > 0 ? units : 1) > 1 ? want / units : 1;
  int64_t chunk = ((span + n - 1) / n + step - 1) / step * step;
  if (chunk < least) chunk = least;
  return Kv8Split{(int)chunk, (int)((span + chunk - 1) / chunk)};
}
// splits that kv8_split never exceeds for any span up to max_len
inline int kv8_most_splits(int max_len, int64_t units, int64_t want, int least) {
  const int64_t n = want / (units > 0 ? units : 1) > 1 ? want / units : 1, m = ((int64_t)max_len + least - 1) / least;
  return (int)(n < m ? n : m);
}

}  // namespace msb
