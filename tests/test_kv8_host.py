"""The 8-bit cache on the host: index arithmetic for right and for broken batches (the kernels' own header, compiled here), the
scales' exponents, and refusals of the C entry points and of the Python mirror (no device is needed for any of them)."""
import ctypes as C
import os
import subprocess

import pytest
import torch

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "macseek_b200", "csrc")

PROGRAM = r"""
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
int main() {
  std::mt19937 rng(5);
  auto upto = [&](int n) { return (int)(rng() % (unsigned)(n + 1)); };
  for (int trial = 0; trial < 4000; trial++) {
    const int shift = 4 + upto(3), block = 1 << shift;
    const int n_seq = upto(9) == 0 ? 1 + upto(2000) : 1 + upto(70), most = upto(3) ? 1 + upto(5) : 1 + upto(400), ctx = upto(1) ? upto(700) : 0;
    std::vector<int> start{0}, len;
    int max_new = 1, max_len = 1;
    for (int s = 0; s < n_seq; s++) {
      const int n = upto(most), l = n + upto(ctx);
      start.push_back(start.back() + n); len.push_back(l);
      max_new = kv8_max(max_new, n); max_len = kv8_max(max_len, l);
    }
    const int n_tokens = kv8_max(start.back() + upto(3), max_new), stride = (max_len + block - 1) / block + upto(2);
    const bool broken = trial % 4 == 3;
    if (broken)
      for (int k = 0; k < 3; k++) {
        const int junk[6] = {-1, -2147483647 - 1, 2147483647, n_tokens + 1, 7, max_len + 1};
        (upto(1) ? start : len)[upto(n_seq - 1)] = junk[upto(5)];
      }
    std::vector<int> seen(n_tokens, 0);
    const int64_t items = kv8_items(n_tokens, n_seq, shift);
    for (int64_t i = 0; i < items; i++) {
      auto first = [&](int s) { NEED(s >= 0 && s < n_seq); return kv8_first_item(start[s], s, shift); };
      const int s = kv8_search(n_seq, (int)i, first, Host());
      NEED(s >= 0 && s < n_seq);
      Kv8Seq q;
      const bool ok = kv8_seq_of(start[s], start[s + 1], len[s], n_tokens, max_new, max_len, q);
      NEED(ok || broken);
      const Kv8Item it = kv8_item_of(q, (int)(i - first(s)), shift);
      if (it.n == 0) continue;
      NEED(it.blk >= 0 && it.blk < stride && it.at >= 0 && it.n > 0 && it.at + it.n <= block);
      NEED(it.row >= 0 && it.row + it.n <= n_tokens);
      NEED(it.blk * block + it.at == q.len - q.n + it.row - q.row);
      for (int r = 0; r < it.n; r++) seen[it.row + r]++;
    }
    if (!broken)
      for (int r = 0; r < n_tokens; r++) NEED(seen[r] == (r < start[n_seq]));
    // the other numbering: as many items for every sequence as the longest needs
    const int each = kv8_touched(max_new, shift);
    std::fill(seen.begin(), seen.end(), 0);
    for (int s = 0; s < n_seq; s++) {
      Kv8Seq q;
      kv8_seq_of(start[s], start[s + 1], len[s], n_tokens, max_new, max_len, q);
      for (int j = 0; j < each; j++) {
        const Kv8Item it = kv8_item_of(q, j, shift);
        NEED(it.n == 0 || (it.blk < stride && it.at + it.n <= block && it.row + it.n <= n_tokens && it.n <= max_new));
        for (int r = 0; r < it.n; r++) seen[it.row + r]++;
      }
    }
    if (!broken)
      for (int r = 0; r < n_tokens; r++) NEED(seen[r] == (r < start[n_seq]));
    // rows -> sequence, key ranges and their splits
    for (int k = 0; k < 20; k++) {
      const int s = upto(n_seq - 1), G = 1 + upto(8), window = upto(1) ? 0 : 1 + upto(300), kvh = 1 + upto(8);
      const bool f32 = upto(1);
      const Kv8Plan pl = kv8_plan(n_seq, max_new, max_len, kvh, kvh * G, 64 << upto(1), f32, window, 148);
      const Kv8Most most = kv8_most(n_seq, max_new, max_len, kvh, kvh * G, f32, 148);
      const int step = pl.step, rows = pl.rows;
      NEED(pl.chunk % step == 0 && pl.chunk > 0 && pl.splits <= (pl.many ? most.many : most.few) && (int64_t)pl.tiles * rows >= (int64_t)max_new * G);
      Kv8Seq q;
      if (!kv8_seq_of(start[s], start[s + 1], len[s], n_tokens, max_new, max_len, q) || q.n == 0) continue;
      if (!broken) {
        const int tok = q.row + upto(q.n - 1);
        NEED(kv8_search(n_seq, tok, [&](int i) { return start[i]; }, Host()) == s);
      }
      for (int m0 = 0; m0 < q.n * G; m0 += rows) {
        const int m1 = kv8_min(m0 + rows, q.n * G);
        const Kv8Range r = kv8_range(q, m0, m1, G, window, step);
        NEED(r.lo >= 0 && r.lo % step == 0 && r.lo < r.hi && r.hi <= q.len);
        for (int m = m0; m < m1; m++) {
          const int pos = q.len - q.n + m / G, from = window ? kv8_max(0, pos - window + 1) : 0;
          NEED(r.lo <= from && pos < r.hi);
        }
        NEED((r.hi - r.lo + pl.chunk - 1) / pl.chunk <= pl.splits);
      }
    }
  }
  puts("ok");
}
"""


def test_index_arithmetic_covers_every_row_once_and_stays_in_bounds(tmp_path):
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(PROGRAM)
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover", "-I" + CSRC, str(src), "-o", str(exe)])
    r = subprocess.run([str(exe)], text=True, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)
    assert r.stdout.strip() == "ok", r.stdout


def test_attention_takes_the_kernel_and_the_split_that_end_sooner(tmp_path):
    # sequences, new rows, tokens, key heads, heads, dim, f32, window -> many rows' kernel, splits of the keys
    cases = {(1, 1, 1, 8, 64, 128, 0, 0): (0, 1), (1, 1, 999, 8, 64, 128, 1, 0): (0, 8), (1, 1, 200000, 8, 64, 128, 0, 0): (0, 55),
             (64, 1, 8192, 8, 64, 128, 0, 0): (0, 4), (64, 1, 8192, 8, 64, 128, 0, 128): (0, 1), (16, 4, 4004, 8, 64, 64, 0, 0): (0, 5),
             (1, 64, 64, 8, 64, 64, 0, 0): (0, 1), (1, 4096, 4096, 8, 64, 128, 0, 0): (1, 1), (1, 4096, 4096, 8, 64, 128, 1, 0): (1, 1),
             (5, 333, 8525, 4, 32, 64, 0, 4096): (1, 1), (1, 256, 1256, 8, 64, 128, 0, 0): (1, 2), (1, 300000, 300000, 8, 64, 64, 0, 16): (1, 1), (1, 16, 16016, 8, 64, 128, 1, 0): (1, 18)}
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text('#include "kv8_index.h"\n#include <cstdio>\nint main() {\n' + "\n".join(
        '{ auto p = msb::kv8_plan(%s, 148); printf("%%d %%d\\n", p.many, p.splits); }' % ", ".join(map(str, c)) for c in cases) + "\n}\n")
    subprocess.check_call(["g++", "-std=c++17", "-I" + CSRC, str(src), "-o", str(exe)])
    got = [tuple(int(v) for v in line.split()) for line in subprocess.check_output([str(exe)], text=True).splitlines()]
    assert dict(zip(cases, got)) == cases


# ------------------------------------------------------------------------------------------------ refusals of the C entry points
BASE = 1 << 20        # an aligned address that nothing follows: every call below is refused before it is used


def _cache(lib, **kw):
    a = dict(n_blocks=4, kv_heads=2, head_dim=64, block=16, k=BASE, v=BASE, k_scale=BASE, v_scale=BASE)
    a.update(kw)
    return lib.Kv8CacheC(*a.values())


def _batch(lib, **kw):
    a = dict(n_seq=2, n_tokens=8, max_new=4, max_len=32, seq_start=BASE, kv_len=BASE, table=BASE, table_stride=2)
    a.update(kw)
    return lib.Kv8BatchC(*a.values())


BAD = [("cache", k, v) for k, v in (("n_blocks", 0), ("kv_heads", 0), ("kv_heads", 2000), ("head_dim", 96), ("block", 48), ("block", 8), ("k", None),
                                    ("v", None), ("k", BASE + 8), ("v_scale", None))] + \
      [("batch", k, v) for k, v in (("n_seq", 0), ("n_seq", 65536), ("n_tokens", 0), ("max_new", 0), ("max_new", 9), ("max_len", 3),
                                    ("max_len", (1 << 30) + 1), ("table_stride", 1), ("seq_start", None), ("kv_len", None), ("table", None))]


@pytest.mark.parametrize("which,key,value", BAD)
def test_entry_points_refuse_bad_caches_and_batches(which, key, value):
    from macseek_b200 import _lib
    c = _cache(_lib, **({key: value} if which == "cache" else {}))
    b = _batch(_lib, **({key: value} if which == "batch" else {}))
    for rc in (_lib.lib.msb_kv8_write(C.byref(c), C.byref(b), 0, BASE, BASE, 128, 128, None),
               _lib.lib.msb_kv8_read(C.byref(c), C.byref(b), 0, BASE, BASE, 128, 128, None),
               _lib.lib.msb_kv8_attn(C.byref(c), C.byref(b), 0, BASE, 256, 4, 0.1, 0, None, BASE, 256, BASE, 1 << 20, None)):
        assert rc == -1 and _lib.lib.msb_last_error()
    assert _lib.lib.msb_kv8_attn_scratch_bytes(C.byref(c), C.byref(b), 4) == 0


def test_entry_points_refuse_bad_rows():
    from macseek_b200 import _lib
    c, b = _cache(_lib), _batch(_lib)
    for call in (_lib.lib.msb_kv8_write, _lib.lib.msb_kv8_read):
        go = lambda ty=0, k=BASE, v=BASE, ks=128, vs=128: call(C.byref(c), C.byref(b), ty, k, v, ks, vs, None)  # noqa: E731
        assert go(ty=8) == -2 and go(k=None) == -1 and go(v=None) == -1 and go(ks=127) == -1 and go(vs=64) == -1
        assert go(k=BASE + 2) == -1 and go(ty=1, v=BASE + 1) == -1
    def attn(ty=0, q=BASE, qs=256, heads=4, scale=0.1, window=0, out=BASE, os=256):
        return _lib.lib.msb_kv8_attn(C.byref(c), C.byref(b), ty, q, qs, heads, scale, window, None, out, os, BASE, 1 << 20, None)
    assert attn(ty=13) == -2 and attn(q=None) == -1 and attn(out=None) == -1 and attn(qs=255) == -1 and attn(os=0) == -1
    assert attn(heads=0) == -1 and attn(heads=3) == -1 and attn(window=-1) == -1
    assert attn(scale=float("nan")) == -1 and attn(scale=float("inf")) == -1 and attn(q=BASE + 1) == -1
    assert _lib.lib.msb_kv8_attn_scratch_bytes(C.byref(c), C.byref(b), 3) == 0


def test_head_norm_rope_refuses():
    from macseek_b200 import _lib

    def go(ty=0, q=BASE, qh=4, qs=256, k=BASE, kh=2, ks=128, n=3, D=64, cs=BASE, pos=BASE, n_pos=9, rot=64, first=0, halves=0, qo=BASE, qos=256,
           ko=BASE, kos=128):
        return _lib.lib.msb_head_norm_rope(ty, q, qh, qs, None, k, kh, ks, None, n, D, 1e-6, cs, pos, n_pos, rot, first, halves, qo, qos, ko, kos, None)
    assert go(ty=2) == -2
    for kw in (dict(q=None), dict(k=None), dict(qo=None), dict(ko=None), dict(qs=255), dict(kos=127), dict(n=0), dict(qh=0, kh=0), dict(qh=-1), dict(kh=32768, ks=1 << 40, kos=1 << 40),
               dict(D=60), dict(D=264), dict(D=0), dict(rot=62), dict(rot=72), dict(rot=-8), dict(first=8), dict(first=-8, rot=32), dict(first=4, rot=32),
               dict(rot=8, halves=1), dict(rot=56, halves=1), dict(pos=None), dict(cs=None), dict(n_pos=0), dict(q=BASE + 2), dict(ty=1, ko=BASE + 1)):
        assert go(**kw) == -1, kw


def test_mirror_refuses_tensors_of_the_host():
    from macseek_b200 import _lib, kv8
    u8, f32, i32 = dict(dtype=torch.uint8), dict(dtype=torch.float32), dict(dtype=torch.int32)
    with pytest.raises(_lib.MsbError):
        kv8.Cache.of(torch.zeros(2, 1, 16, 64, **u8), torch.zeros(2, 1, 16, 64, **u8), torch.ones(2, 1, **f32), torch.ones(2, 1, **f32))
    with pytest.raises(_lib.MsbError):
        kv8.Batch(torch.zeros(2, **i32), torch.zeros(1, **i32), torch.zeros(1, 1, **i32), 1, 1, 1)


class _Stream:
    device = torch.device("cuda", 1)
    device_index = 1


def test_mirror_refuses_another_device_than_the_streams():
    from macseek_b200 import _lib, kv8
    e = type("E", (), {"stream": _Stream()})()
    with pytest.raises(_lib.MsbError, match="stream"):
        kv8._elsewhere(e, torch.device("cuda", 0), None)


@pytest.mark.parametrize("shape,stride,ok", [((3, 2, 64), (128, 64, 1), True), ((3, 2, 64), (400, 64, 1), True), ((1, 2, 64), (9, 64, 1), True),
                                             ((3, 1, 64), (64, 7, 1), True), ((3, 2, 64), (128, 64, 2), False), ((3, 2, 64), (1, 192, 3), False),
                                             ((4, 2, 64), (128, 64, 1), False), ((3, 3, 64), (192, 64, 1), False), ((3, 2, 32), (64, 32, 1), False)])
def test_mirror_takes_rows_with_dense_heads_only(shape, stride, ok):
    from macseek_b200 import _lib, kv8
    t = torch.empty(4096).as_strided(shape, stride)
    want = (shape[0] if ok else 3, shape[1] if ok else 2, 64)
    if ok:
        assert kv8._rows("x", t, *want, t.device) == 0
    else:
        with pytest.raises(_lib.MsbError):
            kv8._rows("x", t, *want, t.device)


def test_mirror_refuses_numbers_beyond_32_bits():
    """Structures and arguments of the C calls are 32-bit: a larger number would arrive as another one."""
    from macseek_b200 import _lib, attn, kv8
    i32 = dict(dtype=torch.int32)
    for bad in ((1 << 32) + 1, 1 << 31, -1):
        for at in range(3):
            sizes = [1, 1, 1]
            sizes[at] = bad
            with pytest.raises(_lib.MsbError, match="32 bits"):
                kv8.Batch(torch.zeros(2, **i32), torch.zeros(1, **i32), torch.zeros(1, 1, **i32), *sizes)
        with pytest.raises(_lib.MsbError, match="32 bits"):
            kv8.attn_scratch(None, None, bad)
        with pytest.raises(_lib.MsbError, match="32 bits"):
            kv8.encode_kv8_attn(None, None, None, None, None, None, window=bad)
        with pytest.raises(_lib.MsbError, match="32 bits"):
            attn.encode_head_norm_rope(None, None, None, None, None, 1e-6, None, None, None, None, rot_first=bad)


@pytest.mark.parametrize("rot,first", [(64, 2147483640), (8, 2147483640), (2147483640, 8), (2147483640, 2147483640)])
def test_head_norm_rope_refuses_dims_whose_sum_passes_32_bits(rot, first):
    from macseek_b200 import _lib
    assert _lib.lib.msb_head_norm_rope(0, BASE, 4, 256, None, BASE, 2, 128, None, 3, 64, 1e-6, BASE, BASE, 9, rot, first, 0, BASE, 256, BASE, 128,
                                       None) == -1
    assert b"rotation" in _lib.lib.msb_last_error()
