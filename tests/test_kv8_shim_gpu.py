"""The 8-bit cache's C++ calls (include/ms_b200_shim.hpp) executed: the same bits as through the mirror."""
import os
import subprocess

import numpy as np
import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def build(tmp_path):
    lib = os.path.join(ROOT, "macseek_b200")
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-Wall", "-I", os.path.join(ROOT, "include"), os.path.join(ROOT, "tests", "kv8_exec.cpp"),
                           "-o", str(tmp_path / "t"), "-L", lib, "-lmacseek_b200", "-Wl,-rpath," + lib, "-L/usr/local/cuda/lib64",
                           "-Wl,-rpath,/usr/local/cuda/lib64"])


def test_compiles_and_links(tmp_path):
    build(tmp_path)


@pytest.mark.gpu
def test_calls_equal_the_mirrors(tmp_path):
    from macseek_b200 import attn, kv8
    from macseek_b200.core import Enc
    n, heads, kvh, dim = 70, 12, 3, 64
    g = torch.Generator().manual_seed(1)
    q, k, v = torch.randn(n, heads, dim, generator=g), torch.randn(n, kvh, dim, generator=g), torch.randn(n, kvh, dim, generator=g)
    qw, kw = 1 + 0.1 * torch.randn(dim, generator=g), 1 + 0.1 * torch.randn(dim, generator=g)
    ang = torch.arange(n)[:, None] * torch.pow(1e4, -torch.arange(dim // 2) * 2.0 / dim)[None]
    cs = torch.stack([ang.cos(), ang.sin()], -1).float().contiguous()
    np.concatenate([t.numpy().reshape(-1) for t in (q, k, v, qw, kw, cs)]).tofile(str(tmp_path / "in"))
    build(tmp_path)
    subprocess.check_call([str(tmp_path / "t"), str(tmp_path / "in"), str(tmp_path / "out")])
    got = torch.from_numpy(np.fromfile(str(tmp_path / "out"), dtype=np.float32))
    q, k, v, qw, kw, cs = (t.cuda() for t in (q, k, v, qw, kw, cs))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    e = Enc()
    attn.encode_head_norm_rope(e, q, k, qw, kw, 1e-6, cs, torch.arange(n, dtype=torch.int32, device="cuda"), q, k, halves=True)
    cache, batch = kv8.Cache(5, kvh, dim, 32), kv8.Batch(i32([0, n]), i32([n]), i32([[4, 0, 2]]), n, n, n)
    kv8.encode_kv8_write(e, cache, batch, k, v)
    ko, vo, out = torch.empty_like(k), torch.empty_like(v), torch.empty_like(q)
    kv8.encode_kv8_read(e, cache, batch, ko, vo)
    kv8.encode_kv8_attn(e, cache, batch, q, out, kv8.attn_scratch(cache, batch, heads), window=40)
    e.wait()
    want = torch.cat([t.cpu().reshape(-1) for t in (out, ko, vo)])
    assert torch.equal(got, want)
