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
      if (p.chunk > kKv8FewKeys) { printf("%d keys in a part\n", p.chunk); return 1; }
    }
  }
  if (few < 1000) { puts("too few cases"); return 1; }
  puts("ok");
}
""")
