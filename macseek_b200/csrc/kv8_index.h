// Index arithmetic of the 8-bit cache's kernels as plain C++, for the kernels and for tests on the host: which rows, blocks and keys a
// block of threads works on, for any contents of a batch's device arrays.  Nothing here gives an index outside what the arguments allow.
#pragma once
#include <algorithm>
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

// In a batch whose starts fall the search above misses items of right sequences.  The next of them from item j of sequence s on, which go on
// behind it (false: none is left).
template <class SeqOf, class Start, class Ballot>
KV8_HD bool kv8_next_missed(int n, int shift, SeqOf seq, Start start, Ballot ballot, int& s, int& j, Kv8Item& it) {
  const auto first = [&](int i) { return kv8_first_item(start(i), i, shift); };
  for (; s < n; s++, j = 0) {
    const Kv8Seq q = seq(s);
    for (;; j++) {
      it = kv8_item_of(q, j, shift);
      if (it.n == 0) break;
      if (kv8_search(n, first(s) + j, first, ballot) != s) { j++; return true; }
    }
  }
  return false;
}

// The sequence that owns row x (-1: none): found by its start, and where starts that fall mislead the search, the first right one that has it.
template <class SeqOf, class Start, class Ballot>
KV8_HD int kv8_owner(int n, int x, SeqOf seq, Start start, Ballot ballot, Kv8Seq& q) {
  int s = kv8_search(n, x, start, ballot);
  q = seq(s);
  if (x >= q.row && x - q.row < q.n) return s;
  for (int s0 = 0; s0 < n; s0 += 32) {
    unsigned m = ballot([&](int lane) {
      if (s0 + lane >= n) return false;
      const Kv8Seq o = seq(s0 + lane);
      return x >= o.row && x - o.row < o.n;
    });
    if (m == 0) continue;
    for (s = s0; !(m & 1); m >>= 1) s++;
    q = seq(s);
    return s;
  }
  return -1;
}

// Keys that rows [m0, m1) of a sequence look at (row r is token r / G of its new ones): [lo, hi), lo being `first` rounded down to `step`.
// Blocks of 16 tokens before `first` need not be there.
struct Kv8Range { int lo, hi, first; };
KV8_HD Kv8Range kv8_range(const Kv8Seq& s, int m0, int m1, int G, int window, int step) {
  const int p0 = s.len - s.n;
  Kv8Range r{0, p0 + (m1 - 1) / G + 1, 0};
  if (window && p0 + m0 / G >= window) {
    r.first = p0 + m0 / G - window + 1;
    r.lo = r.first / step * step;
  }
  return r;
}
// most keys that a tile of `rows` rows looks at, for any sequence
inline int kv8_span(int max_len, int rows, int G, int window, int step) {
  const int64_t w = (int64_t)window + rows / G + 1 + step;
  return window && w < max_len ? (int)w : max_len;
}

// How a call of the attention runs: on the kernel for few rows (blocks of 16 rows of a key head, all of them reading the keys) or on the one
// for many (256, F32 128), and in how many parts the keys are split.  The estimate of a call, in us, from times on a B200: blocks an SM at a
// time, their start, their keys, and for parts the join, which reads what they wrote.  Of sequences whose lengths differ 0.6 are counted.
struct Kv8Plan { int many, rows, step, tiles, chunk, splits; };
constexpr int kKv8FewRows = 16, kKv8FewStep = 32, kKv8ManyRows = 256, kKv8ManyRowsF32 = 128, kKv8ManyStep = 64, kKv8Least = 128;
// Keys whose products a tensor core adds up by itself, cutting off up to 2^-23 of the sum at every 16 keys: in a block of few rows (a part at
// most; a warp has a quarter of them, and of F32 rows it begins anew) and in one of many (then the sum is begun anew).
constexpr int kKv8FewKeys = 65536, kKv8Fold = 16384, kKv8FoldF32 = 1024;
// parts that this takes for few rows (256 at most, 16M tokens: a bound that no sequence comes near shall not cost a scratch and blocks for it)
inline int kv8_least(int keys) { const int n = (int)((keys + kKv8FewKeys - 1ll) / kKv8FewKeys); return n < 256 ? n : 256; }

// splits at most of either kernel, whatever the window
struct Kv8Most { int few, many; };
inline Kv8Most kv8_most(int n_seq, int max_new, int max_len, int kv_heads, int heads, bool f32, int sms) {
  const int64_t rows = (int64_t)max_new * (heads / kv_heads), groups = (int64_t)n_seq * kv_heads, full = (max_len + kKv8Least - 1ll) / kKv8Least;
  const int64_t few = 3ll * sms * (n_seq > 1 ? 6 : 1) / ((rows + kKv8FewRows - 1) / kKv8FewRows * groups);
  const int many_rows = f32 ? kKv8ManyRowsF32 : kKv8ManyRows;
  const int64_t many = 4ll * sms / ((rows + many_rows - 1) / many_rows * groups);
  const int64_t least = kv8_least(max_len);
  return Kv8Most{(int)(few < least ? least : few < full ? few : full), (int)(many < 1 ? 1 : many < full ? many : full)};
}
inline Kv8Plan kv8_plan(int n_seq, int max_new, int max_len, int kv_heads, int heads, int dim, bool f32, int window, int sms) {
  const int G = heads / kv_heads;
  const int64_t rows = (int64_t)max_new * G, groups = (int64_t)n_seq * kv_heads;
  const double part = n_seq > 1 ? 0.6 : 1.0, joined = part * n_seq * max_new * heads * (dim + 2) * 8 / 4e6;      // us a part: written, read
  const auto up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
  const Kv8Most most = kv8_most(n_seq, max_new, max_len, kv_heads, heads, f32, sms);
  double best[2] = {0, 0};
  Kv8Plan plans[2] = {{0, kKv8FewRows, kKv8FewStep, 0, 0, 0}, {1, f32 ? kKv8ManyRowsF32 : kKv8ManyRows, kKv8ManyStep, 0, 0, 0}};
  for (int k = 0; k < 2; k++) {
    Kv8Plan& pl = plans[k];
    const int span = kv8_span(max_len, pl.rows, G, window, pl.step), unit = k ? pl.step : 64, top = k ? most.many : most.few;
    pl.tiles = (int)up(rows, pl.rows);
    const int64_t units = pl.tiles * groups, room = k ? 1 : f32 && dim == 128 ? 2 : 3;      // blocks an SM at once
    // few: keys of 16 rows that an SM does in a us, by all its blocks (one alone: 1 / 1.7 of them); many: us a key of a block's rows
    const double speed = f32 ? (dim == 64 ? 182 : 115) : (dim == 64 ? 230 : 155), per_key = f32 ? (dim == 64 ? 0.032 : 0.044) : (dim == 64 ? 0.031 : 0.034);
    for (int n = k ? 1 : kv8_least(span), last = 0; n <= top; n = n < top ? kv8_min(top, n + kv8_max(1, n / 8)) : top + 1) {
      const int chunk = kv8_max((int)(up(up(span, n), unit) * unit), kKv8Least), parts = (int)up(span, chunk);
      if (parts == last) continue;
      last = parts;
      const int64_t blocks = (int64_t)(units * parts * part) + 1, at_once = std::min(room, up(blocks, sms));
      const double one = k ? 7 + per_key * chunk : 2 + chunk * (at_once > 1 ? at_once : 1.7) / speed;
      const double us = 4 + (double)up(blocks, room * sms) * one + (parts > 1 ? 3 + joined * parts : 0);
      if (pl.splits == 0 || us < best[k]) { best[k] = us; pl.chunk = chunk; pl.splits = parts; }
    }
  }
  return best[0] <= best[1] && (int64_t)plans[0].tiles * kv_heads <= 65535 ? plans[0] : plans[1];     // (of a grid's second dimension)
}

}  // namespace msb
