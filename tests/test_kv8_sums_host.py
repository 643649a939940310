"""Lengths of the attention's sums over the 8-bit cache, and broken batches, in the kernels' own index arithmetic, compiled for the host."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "macseek_b200", "csrc")


def run(tmp_path, program):
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(program)
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover", "-I" + CSRC, str(src), "-o", str(exe)])
    r = subprocess.run([str(exe)], text=True, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)
    assert r.stdout.strip() == "ok", r.stdout


def test_parts_of_few_rows_have_few_enough_keys_for_one_sum(tmp_path):
    run(tmp_path, r"""
#include "kv8_index.h"
#include <cstdio>
#include <random>
using namespace msb;
int main() {
  std::mt19937 rng(1);
  auto upto = [&](int n) { return (int)(rng() % (unsigned)(n + 1)); };
  int few = 0;
  for (int i = 0; i < 20000; i++) {
    const int n_seq = 1 + (upto(2) ? upto(300) : upto(65534)), max_new = 1 + upto(upto(1) ? 3 : 900), max_len = max_new + upto(upto(1) ? 1 << 29 : 300000);
    const int kvh = 1 + upto(15), G = 1 + upto(15), window = upto(1) ? 0 : 1 + upto(400000);
    const bool f32 = upto(1);
    const Kv8Plan p = kv8_plan(n_seq, max_new, max_len, kvh, kvh * G, 64 << upto(1), f32, window, 148);
    const Kv8Most most = kv8_most(n_seq, max_new, max_len, kvh, kvh * G, f32, 148);
    if (p.splits > (p.many ? most.many : most.few) || p.splits < 1 || p.chunk % p.step) { puts("parts"); return 1; }
    const int span = kv8_span(max_len, p.rows, G, window, p.step);
    if ((int64_t)p.chunk * p.splits < span) { puts("keys"); return 1; }
    if (!p.many) {
      few++;
      if (p.chunk > kKv8FewKeys && (span <= 256 * kKv8FewKeys || p.chunk > span / 256 + 64)) { printf("%d keys in a part\n", p.chunk); return 1; }
      if (p.splits > 256 && p.splits > 3 * 148 * 6) { printf("%d parts\n", p.splits); return 1; }
    }
  }
  if (few < 1000) { puts("too few cases"); return 1; }
  puts("ok");
}
""")


BATCH = r"""
#include "kv8_index.h"
#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>
using namespace msb;
static void need(bool ok, const char* what, int line) { if (!ok) { printf("%s (line %d)\n", what, line); exit(1); } }
#define NEED(x) need(x, #x, __LINE__)
struct Host { template <class F> unsigned operator()(F f) const { unsigned m = 0; for (int l = 0; l < 32; l++) if (f(l)) m |= 1u << l; return m; } };
struct Batch {
  std::vector<int> start{0}, len;
  int n_seq, n_tokens, max_new = 1, max_len = 1;
  template <class R> Batch(R& upto, bool broken) {
    n_seq = upto(9) == 0 ? 1 + upto(1500) : 1 + upto(70);
    const int most = upto(3) ? 1 + upto(5) : 1 + upto(400), ctx = upto(1) ? upto(700) : 0;
    for (int s = 0; s < n_seq; s++) {
      const int n = upto(most), l = n + upto(ctx);
      start.push_back(start.back() + n); len.push_back(l);
      max_new = kv8_max(max_new, n); max_len = kv8_max(max_len, l);
    }
    n_tokens = kv8_max(start.back() + upto(3), max_new);
    if (broken)
      for (int k = 0; k < 1 + upto(3); k++) {
        const int junk[7] = {-1, -2147483647 - 1, 2147483647, n_tokens + 1, 7, max_len + 1, upto(n_tokens)};
        if (upto(3)) start[upto(n_seq)] = junk[upto(6)];
        else len[upto(n_seq - 1)] = junk[upto(6)];
      }
  }
  Kv8Seq seq(int s) const {
    Kv8Seq q;
    kv8_seq_of(start[s], start[s + 1], len[s], n_tokens, max_new, max_len, q);
    return q;
  }
};
"""


def test_every_row_of_a_right_sequence_has_an_owner_in_broken_batches(tmp_path):
    run(tmp_path, BATCH + r"""
int main() {
  std::mt19937 rng(7);
  auto upto = [&](int n) { return (int)(rng() % (unsigned)(n + 1)); };
  for (int trial = 0; trial < 3000; trial++) {
    const Batch b(upto, trial % 4 != 0);
    std::vector<int> owners(b.n_tokens, 0);
    for (int s = 0; s < b.n_seq; s++) { const Kv8Seq q = b.seq(s); for (int i = 0; i < q.n; i++) owners[q.row + i]++; }
    for (int k = 0; k < 200; k++) {
      const int x = upto(b.n_tokens - 1);
      Kv8Seq q;
      const int s = kv8_owner(b.n_seq, x, [&](int i) { NEED(i >= 0 && i < b.n_seq); return b.seq(i); }, [&](int i) { return b.start[i]; }, Host(), q);
      NEED((s >= 0) == (owners[x] > 0));
      if (s < 0) continue;
      const Kv8Seq o = b.seq(s);
      NEED(o.row == q.row && o.n == q.n && o.len == q.len && x >= o.row && x < o.row + o.n);
    }
  }
  puts("ok");
}
""")


def test_every_item_of_a_right_sequence_is_done_once_in_broken_batches(tmp_path):
    run(tmp_path, BATCH + r"""
int main() {
  std::mt19937 rng(9);
  auto upto = [&](int n) { return (int)(rng() % (unsigned)(n + 1)); };
  int missed = 0;
  for (int trial = 0; trial < 2000; trial++) {
    const bool broken = trial % 4 != 0;
    const Batch b(upto, broken);
    const int shift = 4 + upto(3);
    auto seq = [&](int i) { NEED(i >= 0 && i < b.n_seq); return b.seq(i); };
    auto start = [&](int i) { NEED(i >= 0 && i <= b.n_seq); return b.start[i]; };
    auto first = [&](int i) { return kv8_first_item(start(i), i, shift); };
    std::vector<std::vector<int>> done(b.n_seq);
    for (int s = 0; s < b.n_seq; s++) done[s].assign(b.seq(s).n, 0);
    auto work = [&](int s, const Kv8Item& it) {
      const Kv8Seq q = b.seq(s);
      NEED(it.row >= q.row && it.row + it.n <= q.row + q.n && it.blk * (1 << shift) + it.at == q.len - q.n + it.row - q.row);
      for (int r = 0; r < it.n; r++) done[s][it.row - q.row + r]++;
    };
    const int64_t items = kv8_items(b.n_tokens, b.n_seq, shift);
    for (int64_t x = 0; x < items; x++) {
      const int s = kv8_search(b.n_seq, (int)x, first, Host());
      const Kv8Item it = kv8_item_of(b.seq(s), (int)x - first(s), shift);
      if (it.n) work(s, it);
    }
    int s = 0, j = 0;
    Kv8Item it;
    while (kv8_next_missed(b.n_seq, shift, seq, start, Host(), s, j, it)) { NEED(broken); missed++; work(s, it); }
    for (auto& d : done) for (int n : d) NEED(n == 1);
    bool falls = false;                                              // where no start falls nothing is missed, whatever else is wrong
    for (int i = 0; i < b.n_seq; i++) falls |= b.start[i + 1] < b.start[i];
    if (!falls) { s = j = 0; NEED(!kv8_next_missed(b.n_seq, shift, seq, start, Host(), s, j, it)); }
  }
  NEED(missed > 1000);
  puts("ok");
}
""")
