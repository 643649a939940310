"""Grouped-query heads over the 8-bit cache: head norms with rotation, writing, reading and attention against 64 bits."""
import pytest
import torch

import kv8_ref as R

pytestmark = pytest.mark.gpu


def enc(stream=None):
    from macseek_b200.core import Enc
    return Enc(stream)


def spread(t, extra=24, shift=0):
    """The same rows inside wider ones, `shift` elements off."""
    n, h, d = t.shape
    buf = torch.full((n * (h * d + extra) + shift + 8,), 7.0, dtype=t.dtype, device=t.device)
    v = buf[shift:shift + n * (h * d + extra)].view(n, h * d + extra)[:, :h * d].unflatten(1, (h, d))
    v.copy_(t)
    return v, buf


# ------------------------------------------------------------------------------------------------ head norms with rotation
NR = [(1, 64, 8, 128, 64, 64, False, "f32"), (1, 8, 1, 64, 64, 0, True, "bf16"), (37, 32, 4, 64, 32, 0, True, "f16"), (5, 7, 3, 96, 64, 32, False, "f32"),
      (9, 3, 1, 256, 256, 0, True, "bf16"), (2, 1, 1, 8, 8, 0, False, "f32"), (3, 5, 2, 80, 48, 16, True, "f16"), (1100, 6, 2, 128, 128, 0, True, "bf16"),
      (4, 2, 2, 128, 0, 0, False, "f32"), (1030, 40, 8, 64, 64, 0, False, "f32"), (6, 4, 4, 192, 16, 8, True, "bf16")]


@pytest.mark.parametrize("n,qh,kh,D,rot,first,halves,dt", NR)
@pytest.mark.parametrize("form", ("dense", "wide", "odd", "inplace", "no weights"))
def test_head_norm_rope(n, qh, kh, D, rot, first, halves, dt, form):
    from macseek_b200 import attn
    g = torch.Generator().manual_seed(n + D + rot)
    rnd = lambda *s: torch.randn(s, generator=g)  # noqa: E731
    q, k = (3 * rnd(n, qh, D)).to(R.DT[dt]).cuda(), (rnd(n, kh, D) * 0.01).to(R.DT[dt]).cuda()
    q[0, 0] = 0                                                     # a head of zeros
    qw, kw = (None, None) if form == "no weights" else ((1 + 0.3 * rnd(D)).cuda(), (1 + 0.3 * rnd(D)).cuda())
    ang = torch.arange(50, dtype=torch.float64)[:, None] * torch.pow(1e4, -torch.arange(rot // 2) / max(rot // 2, 1))[None]
    cs = torch.stack([ang.cos(), ang.sin()], -1).float().reshape(50, rot // 2, 2).contiguous().cuda()
    pos = torch.randint(0, 50, (n,), generator=g, dtype=torch.int32).cuda()
    if n > 2:
        pos[1] = -1                                                 # padding
    want = [R.norm_rope_ref(q, qw, 1e-6, cs, pos, first, halves), R.norm_rope_ref(k, kw, 1e-6, cs, pos, first, halves)]
    bufs = []
    if form in ("wide", "odd"):
        shift = 0 if form == "wide" else 1
        (q, _), (k, _) = spread(q, 24, shift), spread(k, 8, shift)
        (qo, b0), (ko, b1) = spread(torch.full_like(q, 7), 16, shift), spread(torch.full_like(k, 7), 40, shift)
        bufs = [b0, b1]
    elif form == "inplace":
        qo, ko = q, k
    else:
        qo, ko = torch.full((n, qh, D), 7.0, dtype=q.dtype, device="cuda"), torch.full((n, kh, D), 7.0, dtype=q.dtype, device="cuda")
    kept = [qo.clone(), ko.clone()]
    e = enc()
    attn.encode_head_norm_rope(e, q, k, qw, kw, 1e-6, cs, pos, qo, ko, rot_first=first, halves=halves)
    e.wait()
    half, tiny = R.half_step(q.dtype)
    for got, (ref, tol), was in zip((qo, ko), want, kept):
        live = (pos >= 0)
        assert torch.equal(got[~live], was[~live])
        assert ((got.double() - ref).abs() <= tol * (1 + half) + half * ref.abs() + tiny)[live].all()
    for b in bufs:                                                  # nothing between the rows is touched
        assert int((b == 7).sum()) >= 8
        m = torch.ones_like(b, dtype=torch.bool)
        for t in (qo, ko):
            if t.untyped_storage().data_ptr() == b.untyped_storage().data_ptr():
                m.as_strided(t.shape, t.stride(), t.storage_offset()).fill_(False)
        assert (b[m] == 7).all()


def test_head_norm_rope_of_one_side_and_positions_beyond_the_table():
    from macseek_b200 import _lib, attn
    e = enc()
    q = torch.randn(4, 3, 64, device="cuda")
    cs = torch.randn(10, 32, 2, device="cuda")
    pos = torch.tensor([0, 10, -3, 9], dtype=torch.int32, device="cuda")
    out = torch.full_like(q, 7)
    attn.encode_head_norm_rope(e, q, None, None, None, 1e-6, cs, pos, out, None)
    torch.cuda.synchronize()
    assert _lib.device_status() == 4
    ref, tol = R.norm_rope_ref(q, None, 1e-6, cs, pos.clamp(0, 9), 0, False)
    for r in (0, 3):
        assert ((out[r].double() - ref[r]).abs() <= tol[r] + ref[r].abs() * 2.0 ** -24).all()
    assert (out[1:3] == 7).all()
    out.fill_(7)
    attn.encode_head_norm_rope(e, None, q, None, None, 1e-6, cs, pos.clamp(0, 9), None, out)
    e.wait()
    assert ((out.double() - ref).abs() <= tol + ref.abs() * 2.0 ** -24).all()


# ------------------------------------------------------------------------------------------------ writing and reading
WR = [([(1, 1)], 1, 64, 16), ([(1, 17), (1, 16), (1, 64), (1, 65)], 8, 128, 64), ([(5, 5), (0, 9), (64, 64), (130, 200), (1, 128)], 2, 64, 64),
      ([(300, 1000), (16, 32), (33, 47)], 3, 128, 128), ([(17, 17)] * 40, 1, 64, 32), ([(0, 0), (2, 65), (0, 3), (63, 127)], 4, 128, 16),
      ([(1, 1 + i) for i in range(70)], 2, 64, 16)]


@pytest.mark.parametrize("seqs,heads,dim,block", WR)
@pytest.mark.parametrize("dt", ("f32", "f16", "bf16"))
def test_write_and_read(seqs, heads, dim, block, dt):
    from macseek_b200 import kv8
    c = R.Case(seqs, heads, dim, block, seed=len(seqs) + dim, pad=3)
    mul = 2.0 ** torch.randint(-6, 7, (c.rows, heads, 1), generator=c.g).to(R.DT[dt]).cuda()
    k, v = c.randn(c.rows, heads, dim, dt=dt) * mul, c.randn(c.rows, heads, dim, dt=dt)
    v[:, 0] = 0                                                      # blocks of zeros
    k[c.start_host[-1]:] = float("nan")                              # padding
    k, _ = spread(k, 8 if dt == "f32" else 3)
    want = R.write_ref(c, k, v)
    before = [t.clone() for t in (c.k, c.v)]
    e = enc()
    cache, batch = c.cache(), c.batch()
    kv8.encode_kv8_write(e, cache, batch, k, v)
    e.wait()
    touched = torch.zeros(c.k.shape[0], c.block, dtype=torch.bool, device="cuda")      # rows that a write may change
    for s, (n, l) in enumerate(seqs):
        for p in range((l - n) // block * block, l if n else 0):
            touched[int(c.table_host[s, p // block]), p % block] = True
    for codes, scale, was, val, sc in ((c.k, c.ks, before[0], want[0], want[1]), (c.v, c.vs, before[1], want[2], want[3])):
        m = touched[:, None, :, None].expand_as(codes)
        assert torch.equal(codes[~m], was[~m])
        assert torch.equal(R.values(codes)[m], val[m])
        assert torch.equal(scale.double().nan_to_num(-1), sc.nan_to_num(-1))
    # the rows written, and whole sequences, read back
    for full in (False, True):
        if full:
            c2 = R.Case(seqs, heads, dim, block, seed=1)
            c2.seqs = [(l, l) for _, l in seqs]
            import numpy as np
            st = np.cumsum([0] + [l for _, l in seqs])
            c2.start_host, c2.rows = [int(x) for x in st], int(st[-1]) + 2
            c2.start = torch.tensor(st, dtype=torch.int32, device="cuda")
            c2.max_new = c2.max_len = c.max_len
            c2.len, c2.table, c2.table_host, c2.k, c2.v, c2.ks, c2.vs = c.len, c.table, c.table_host, c.k, c.v, c.ks, c.vs
        else:
            c2 = c
        for shift in (0, 1):
            (ko, kb), (vo, vb) = (spread(torch.full((c2.rows, heads, dim), 7.0, dtype=R.DT[dt], device="cuda"), 16, shift) for _ in range(2))
            kv8.encode_kv8_read(e, cache, c2.batch(), ko, vo)
            e.wait()
            for which, out in (("k", ko), ("v", vo)):
                for s, (n, l) in enumerate(c2.seqs):
                    r = slice(c2.start_host[s], c2.start_host[s] + n)
                    assert torch.equal(out[r], c2.held(s, which, l - n).transpose(0, 1).float().to(R.DT[dt]))
                assert (out[c2.start_host[-1]:] == 7).all()
            for b, t in ((kb, ko), (vb, vo)):
                m = torch.ones_like(b, dtype=torch.bool)
                m.as_strided(t.shape, t.stride(), t.storage_offset()).fill_(False)
                assert (b[m] == 7).all()


def test_write_token_by_token_moves_older_codes_to_a_growing_scale():
    from macseek_b200 import kv8
    heads, dim, block = 2, 64, 16
    c = R.Case([(1, 1)], heads, dim, block, seed=3)
    e = enc()
    cache = kv8.Cache(3, heads, dim, block)
    c.k, c.v, c.ks, c.vs = cache.k, cache.v, cache.k_scale, cache.v_scale
    c.table_host = torch.tensor([[2, 0, 1]])
    c.table = c.table_host.int().cuda()
    for p in range(40):
        c.seqs = [(1, p + 1)]
        c.len = torch.tensor([p + 1], dtype=torch.int32, device="cuda")
        c.max_len = p + 1
        x = c.randn(1, heads, dim) * 2.0 ** (p % 16 - 8)
        want = R.write_ref(c, x, -x)
        kv8.encode_kv8_write(e, cache, c.batch(), x, -x)
        e.wait()
        assert torch.equal(R.values(c.k), want[0]) and torch.equal(R.values(c.v), want[2])
        assert torch.equal(c.ks.double(), want[1]) and torch.equal(c.vs.double(), want[3])


@pytest.mark.parametrize("dt", ("f32", "f16", "bf16"))
def test_write_of_ends_of_the_range(dt):
    """Values at the border of a scale, the smallest and largest numbers, infinities; a NaN is said."""
    from macseek_b200 import _lib, kv8
    dim, block = 64, 16
    big = float(torch.finfo(R.DT[dt]).max)
    rows = torch.zeros(6 * 16, 1, dim)
    for i, top in enumerate((448.0, 448.5 if dt == "f32" else 450.0, 2.0 ** -14, big, float("inf"), 0.875)):
        rows[16 * i:16 * i + 16] = torch.randn(16, 1, dim, generator=torch.Generator().manual_seed(i)).clamp(-1, 1) * min(top, big) * 0.5
        rows[16 * i + 3, 0, 5] = top
        rows[16 * i + 4, 0, 6] = -top
    if dt == "f32":
        rows[0, 0, 0] = 1e-45
        rows[40] = 3e-39
    k = rows.to(R.DT[dt]).cuda()
    c = R.Case([(16, 16)] * 6, 1, dim, block, seed=1)
    want = R.write_ref(c, k, -k)
    e = enc()
    kv8.encode_kv8_write(e, c.cache(), c.batch(), k, -k)
    e.wait()
    for s in range(6):
        b = int(c.table_host[s, 0])
        assert torch.equal(R.values(c.k)[b], want[0][b]) and torch.equal(R.values(c.v)[b], want[2][b])
        assert float(c.ks[b]) == float(want[1][b]) and float(c.vs[b]) == float(want[3][b])
    k[17, 0, 9] = float("nan")
    want = R.write_ref(c, k, -k)
    kv8.encode_kv8_write(e, c.cache(), c.batch(), k, -k)
    torch.cuda.synchronize()
    assert _lib.device_status() == 5
    b = int(c.table_host[1, 0])
    assert torch.equal(R.values(c.k)[b], want[0][b]) and not torch.isnan(R.values(c.v)[b]).any()


# ------------------------------------------------------------------------------------------------ attention
LENS = [[(1, 1)], [(1, 15), (1, 16), (1, 17)], [(1, 63), (1, 64), (1, 65), (1, 1000)], [(4, 4), (2, 130), (0, 50), (3, 77)], [(1, 2500)]]


def check_attn(c, q, out, was, scale, window, sinks):
    ref, tol = R.attn_ref(c, q, was, scale, window, sinks)
    end = c.start_host[-1]
    assert torch.equal(out[end:], was[end:])                         # padding rows stay
    d = (out.double() - ref).abs()
    assert (d <= tol).all(), (float(d.max()), float((d / tol.clamp(min=1e-300))[:end].max()))


@pytest.mark.parametrize("seqs", LENS)
@pytest.mark.parametrize("kv_heads,G,dim,block", [(1, 1, 64, 16), (2, 8, 128, 64), (3, 5, 128, 16), (2, 7, 64, 128), (1, 40, 64, 32)])
@pytest.mark.parametrize("dt", ("f32", "f16", "bf16"))
def test_attention_of_few_rows(seqs, kv_heads, G, dim, block, dt):
    from macseek_b200 import kv8
    c = R.Case(seqs, kv_heads, dim, block, seed=dim + G, pad=2)
    heads, scale = kv_heads * G, dim ** -0.5
    e = enc()
    cache, batch = c.cache(), c.batch()
    scratch = kv8.attn_scratch(cache, batch, heads)
    for window, sink, shift in ((0, False, 0), (0, True, 1), (20, False, 0), (1, True, 0), (700, False, 1)):
        q, _ = spread(c.randn(c.rows, heads, dim, dt=dt, mul=3.0), 24, shift)
        out, _ = spread(torch.full((c.rows, heads, dim), 7.0, dtype=R.DT[dt], device="cuda"), 8, shift)
        was = out.clone()
        sinks = c.randn(heads, mul=2.0) if sink else None
        scratch.fill_(255)
        kv8.encode_kv8_attn(e, cache, batch, q, out, scratch, window=window, sinks=sinks)
        e.wait()
        check_attn(c, q, out, was, scale, window, sinks)


CHUNKS = [[(128, 128)], [(129, 129), (127, 300)], [(33, 33), (1, 500), (0, 20), (300, 700)], [(64, 5000)], [(1000, 1000)], [(17, 2049), (65, 65)]]


@pytest.mark.parametrize("seqs", CHUNKS)
@pytest.mark.parametrize("kv_heads,G,dim,block", [(2, 8, 128, 64), (1, 1, 64, 16), (3, 5, 128, 16), (2, 7, 64, 128), (1, 16, 64, 32), (1, 130, 128, 64)])
@pytest.mark.parametrize("dt", ("f32", "f16", "bf16"))
def test_attention_of_many_rows(seqs, kv_heads, G, dim, block, dt):
    from macseek_b200 import kv8
    if G == 130:
        seqs = [(min(n, 3), l) for n, l in seqs]                     # one token is more than a tile of rows
    c = R.Case(seqs, kv_heads, dim, block, seed=dim + G, pad=2)
    heads, scale = kv_heads * G, dim ** -0.5
    e = enc()
    cache, batch = c.cache(), c.batch()
    scratch = kv8.attn_scratch(cache, batch, heads)
    for window, sink, shift, sc in ((0, False, 0, scale), (0, True, 1, scale), (50, False, 0, -scale), (1, True, 0, 2 * scale), (300, False, 1, scale)):
        q, _ = spread(c.randn(c.rows, heads, dim, dt=dt, mul=3.0), 24, shift)
        out, _ = spread(torch.full((c.rows, heads, dim), 7.0, dtype=R.DT[dt], device="cuda"), 8, shift)
        was = out.clone()
        sinks = c.randn(heads, mul=2.0) if sink else None
        scratch.fill_(255)
        kv8.encode_kv8_attn(e, cache, batch, q, out, scratch, scale=sc, window=window, sinks=sinks)
        e.wait()
        check_attn(c, q, out, was, sc, window, sinks)


@pytest.mark.parametrize("dt", ("f32", "bf16"))
@pytest.mark.parametrize("dim", (64, 128))
def test_attention_over_blocks_of_very_different_scales(dt, dim):
    """Weights carry the blocks' value scales: neither a small one next to a large one nor the largest and smallest lose anything."""
    from macseek_b200 import kv8
    c = R.Case([(1, 200), (3, 120), (40, 200)], 1, dim, 16, seed=2)
    for spread_v in (20, 35, 50):                                   # the widest that a cache has
        c.vs.copy_(torch.exp2(torch.randint(-spread_v, spread_v + 1, c.vs.shape, generator=c.g).float()))
        c.ks.copy_(torch.exp2(torch.randint(-14, -5, c.ks.shape, generator=c.g).float()))
        cache, batch = c.cache(), c.batch()
        q, out = c.randn(c.rows, 4, dim, dt=dt, mul=0.1), torch.zeros(c.rows, 4, dim, dtype=R.DT[dt], device="cuda")
        e = enc()
        kv8.encode_kv8_attn(e, cache, batch, q, out, kv8.attn_scratch(cache, batch, 4))
        e.wait()
        check_attn(c, q, out, out, dim ** -0.5, 0, None)


@pytest.mark.parametrize("seqs,kv_heads,G", [([(1, 1000), (1, 3)], 2, 8), ([(1, 260)], 8, 8), ([(3, 900), (0, 700), (2, 129), (1, 1)], 1, 20),
                                             ([(4, 1024)], 4, 4), ([(1, 128), (1, 129), (1, 640)], 3, 1)])
@pytest.mark.parametrize("dt", ("f32", "bf16"))
@pytest.mark.parametrize("dim", (64, 128))
def test_attention_whose_parts_are_a_cluster(seqs, kv_heads, G, dim, dt):
    """Few rows over a few hundred keys: parts without keys among them, and rows that are not there."""
    from macseek_b200 import kv8
    c = R.Case(seqs, kv_heads, dim, 32, seed=G, pad=1)
    cache, batch, e = c.cache(), c.batch(), enc()
    for window, sink in ((0, True), (100, False), (300, True)):
        q = c.randn(c.rows, kv_heads * G, dim, dt=dt, mul=3.0)
        out = torch.full_like(q, 7)
        sinks = c.randn(kv_heads * G) if sink else None
        kv8.encode_kv8_attn(e, cache, batch, q, out, kv8.attn_scratch(cache, batch, kv_heads * G), window=window, sinks=sinks)
        e.wait()
        check_attn(c, q, out, torch.full_like(q, 7), dim ** -0.5, window, sinks)


def test_attention_results_do_not_depend_on_the_run_or_on_neighbours():
    from macseek_b200 import kv8
    c = R.Case([(1, 900), (1, 3000), (2, 64)], 2, 128, 64, seed=5)
    q = c.randn(c.rows, 16, 128, dt="bf16")
    cache, batch, e = c.cache(), c.batch(), enc()
    outs = []
    for _ in range(3):
        out = torch.zeros_like(q)
        kv8.encode_kv8_attn(e, cache, batch, q, out, kv8.attn_scratch(cache, batch, 16))
        outs.append(out)
    e.wait()
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_broken_batches_are_left_out_and_said():
    """Numbers that cannot be right: that sequence is left out, the others are computed; a block that is not there is not seen."""
    from macseek_b200 import _lib, kv8
    e = enc()

    def make():
        return R.Case([(2, 40), (1, 33), (3, 50)], 2, 64, 16, seed=9)
    for key, at, value in (("len", 1, -4), ("len", 1, 10 ** 6), ("len", 1, 0), ("start", 1, 100), ("start", 1, -2)):
        c = make()
        getattr(c, key)[at] = value
        cache, batch = c.cache(), c.batch()
        q = c.randn(c.rows, 4, 64)
        out = torch.full_like(q, 7)
        kv8.encode_kv8_attn(e, cache, batch, q, out, kv8.attn_scratch(cache, batch, 4))
        torch.cuda.synchronize()
        assert _lib.device_status() == 4
        ref, tol = R.attn_ref(c, q, out, 0.125)
        good = slice(3, 6) if key == "len" else slice(3, 6)
        assert ((out.double() - ref).abs() <= tol)[good].all()
        if key == "len":
            assert (out[2] == 7).all()
            assert ((out.double() - ref).abs() <= tol)[:2].all()
        k = c.randn(c.rows, 2, 64)
        kv8.encode_kv8_write(e, cache, batch, k, k)
        torch.cuda.synchronize()
        assert _lib.device_status() == 4
        kv8.encode_kv8_read(e, cache, batch, k, k.clone())
        torch.cuda.synchronize()
        assert _lib.device_status() == 4
    c = make()
    full = c.table_host.clone()
    c.table[2, 1] = -7                                                # tokens 16 .. 31 of the last sequence
    cache, batch = c.cache(), c.batch()
    q = c.randn(c.rows, 4, 64)
    out = torch.zeros_like(q)
    kv8.encode_kv8_attn(e, cache, batch, q, out, kv8.attn_scratch(cache, batch, 4))
    torch.cuda.synchronize()
    assert _lib.device_status() == 4
    k, v = c.held(2, "k"), c.held(2, "v")
    there = torch.tensor([p < 16 or p >= 32 for p in range(50)], device="cuda")
    for i in range(3):
        m = there & (torch.arange(50, device="cuda") <= 47 + i)
        for h in range(4):
            lg = (k[h // 2] @ q[3 + i, h].double() * 0.125).masked_fill(~m, -torch.inf)
            assert ((torch.softmax(lg, 0) @ v[h // 2]) - out[3 + i, h].double()).abs().max() < 1e-4
    c.table[2] = 999
    out.fill_(7)
    kv8.encode_kv8_attn(e, cache, batch, q, out, kv8.attn_scratch(cache, batch, 4))
    torch.cuda.synchronize()
    assert _lib.device_status() == 4
    assert (out[3:] == 0).all()                                       # rows that see nothing
    ko, vo = torch.full((c.rows, 2, 64), 7.0, device="cuda"), torch.full((c.rows, 2, 64), 7.0, device="cuda")
    kv8.encode_kv8_read(e, cache, batch, ko, vo)
    torch.cuda.synchronize()
    assert _lib.device_status() == 4 and (ko[3:] == 0).all() and (vo[3:] == 0).all() and not (ko[:3] == 7).any()
    was = c.k.clone()
    kv8.encode_kv8_write(e, cache, c.batch(), ko, vo)
    torch.cuda.synchronize()
    assert _lib.device_status() == 4
    kept = [int(i) for i in full[2, :4]]
    assert torch.equal(c.k[kept], was[kept])


def test_refusals_that_need_a_device():
    from macseek_b200 import _lib, kv8
    c = R.Case([(1, 5000)], 2, 128, 64, seed=1)
    cache, batch = c.cache(), c.batch()
    q = c.randn(c.rows, 16, 128)
    e = enc()
    small = torch.empty(64, dtype=torch.uint8, device="cuda")
    with pytest.raises(_lib.MsbError, match="scratch"):
        kv8.encode_kv8_attn(e, cache, batch, q, torch.empty_like(q), small)
    with pytest.raises(_lib.MsbError):
        kv8.encode_kv8_attn(e, cache, batch, q, torch.empty_like(q).half(), kv8.attn_scratch(cache, batch, 16))
    with pytest.raises(_lib.MsbError):
        kv8.encode_kv8_attn(e, cache, batch, q.cpu(), torch.empty_like(q), kv8.attn_scratch(cache, batch, 16))
    with pytest.raises(_lib.MsbError):
        kv8.attn_scratch(cache, batch, 15)
    with pytest.raises((_lib.MsbError, RuntimeError)):               # no strides to ask for: refused, not ended
        kv8.encode_kv8_attn(e, cache, batch, q.to_sparse(), torch.empty_like(q), kv8.attn_scratch(cache, batch, 16))
    with pytest.raises(_lib.MsbError):
        kv8.encode_kv8_write(e, cache, batch, c.randn(c.rows, 2, 128), c.randn(c.rows, 2, 128).half())
    with pytest.raises(_lib.MsbError):
        kv8.encode_kv8_read(e, cache, batch, c.randn(c.rows, 2, 64), c.randn(c.rows, 2, 128))
    with pytest.raises(_lib.MsbError, match="sinks"):
        kv8.encode_kv8_attn(e, cache, batch, q, torch.empty_like(q), kv8.attn_scratch(cache, batch, 16), sinks=torch.zeros(15, device="cuda"))
    from macseek_b200 import attn
    cs, pos = torch.zeros(9, 32, 2, device="cuda"), torch.zeros(c.rows, dtype=torch.int32, device="cuda")
    for bad in (dict(q=q.cpu()), dict(q_w=torch.ones(64, device="cuda")), dict(pos=pos.long()), dict(cs=cs[:, :, 0]), dict(q_out=q.half())):
        a = dict(q=q, q_w=None, pos=pos, cs=cs, q_out=torch.empty_like(q))
        a.update(bad)
        with pytest.raises(_lib.MsbError):
            attn.encode_head_norm_rope(e, a["q"], None, a["q_w"], None, 1e-6, a["cs"], a["pos"], a["q_out"], None)
    e.wait()


def test_scratch_that_is_not_one_piece_of_memory_is_refused():
    """Elements of an expanded or strided tensor are not the bytes behind its pointer."""
    from macseek_b200 import _lib, kv8
    c = R.Case([(1, 5000)], 2, 128, 64, seed=1)
    cache, batch = c.cache(), c.batch()
    q = c.randn(c.rows, 16, 128)
    e, out = enc(), torch.empty_like(q)
    whole = kv8.attn_scratch(cache, batch, 16)
    for bad in (whole[:1].expand(whole.numel()), torch.empty(2 * whole.numel(), dtype=torch.uint8, device="cuda")[::2]):
        with pytest.raises(_lib.MsbError, match="contiguous"):
            kv8.encode_kv8_attn(e, cache, batch, q, out, bad)
    kv8.encode_kv8_attn(e, cache, batch, q, out, whole)
    e.wait()


@pytest.mark.parametrize("dt", ("f32", "bf16"))
@pytest.mark.parametrize("n", (1, 64))
def test_attention_where_the_largest_logit_comes_late_or_is_huge(n, dt):
    """Logits that grow along the keys by far more than a weight may grow before the sums are rescaled, and ones of 1e6 and more."""
    from macseek_b200 import kv8
    D = 64
    c = R.Case([(n, 700)], 1, D, 64, seed=4)
    c.k.fill_(0x38)                                                   # ones
    cache, batch, e = c.cache(), c.batch(), enc()
    q = torch.full((c.rows, 4, D), 1.0, dtype=R.DT[dt], device="cuda") * torch.tensor([1.0, -1.0, 0.5, 0.0], device="cuda", dtype=R.DT[dt])[None, :, None]
    for first, factor in ((1, 2.0), (2.0 ** 20, 1.0), (1, 8.0)):
        for b in range(11):                                           # key scales: a block's logits are first * factor^b * 64 * scale
            c.ks[c.table_host[0, b]] = first * factor ** b
        out = torch.zeros_like(q)
        kv8.encode_kv8_attn(e, cache, batch, q, out, kv8.attn_scratch(cache, batch, 4))
        e.wait()
        assert not torch.isnan(out).any()
        # a row of equal keys inside each block: the average over the last block it sees (positive), the first (negative) or all (zero)
        ref, _ = R.attn_ref(c, q, out, D ** -0.5)
        half, _ = R.half_step(q.dtype)
        # equal keys have equal weights: what is left is the weights' rounding, their sum and the output's
        tol = 4.0 * (2.0 ** -11 + 700 / 8 * 2.0 ** -23 + 2.0 ** -20 + 700 * 2.0 ** -25 + half)
        assert float((out.double() - ref).abs().max()) <= tol * float(c.held(0, "v").abs().max()) / 4


def test_attention_of_what_is_not_a_number_ends():
    """NaN, infinite and absurdly large queries: the call ends, and rows beside them are not touched by them."""
    from macseek_b200 import kv8
    for n in (1, 80):
        c = R.Case([(n, 300), (n, 200)], 1, 64, 16, seed=6)
        q = c.randn(c.rows, 4, 64)
        q[0, 0, 3], q[0, 1, 5], q[0, 2] = float("nan"), float("inf"), 1e38
        cache, batch, e = c.cache(), c.batch(), enc()
        out = torch.zeros_like(q)
        kv8.encode_kv8_attn(e, cache, batch, q, out, kv8.attn_scratch(cache, batch, 4))
        e.wait()
        assert torch.isnan(out[0, 0]).all()
        q[0, :3] = 0
        ref, tol = R.attn_ref(c, q, out, 0.125)
        bad = (out.double() - ref).abs() > tol
        bad[0, :3] = False
        assert not bad.any()


# ------------------------------------------------------------------------------------------------ as they are used
class Model:
    """The attention of one layer as an engine runs it: head norms and rotation, the cache, attention; and the same in 64 bits on what the
    cache holds."""

    def __init__(self, heads, kv_heads, dim, block, dt, seqs, blocks_each, seed=0):
        from macseek_b200 import kv8
        self.heads, self.kv_heads, self.dim, self.block, self.dt = heads, kv_heads, dim, block, R.DT[dt]
        self.g = torch.Generator().manual_seed(seed)
        self.cache = kv8.Cache(seqs * blocks_each + 1, kv_heads, dim, block)
        self.table_host = (torch.randperm(seqs * blocks_each, generator=self.g) + 1).reshape(seqs, blocks_each)
        self.table = self.table_host.int().cuda()
        self.qw, self.kw = ((1 + 0.2 * torch.randn(dim, generator=self.g)).cuda() for _ in range(2))
        ang = torch.arange(4096, dtype=torch.float64)[:, None] * torch.pow(1e4, -torch.arange(dim // 2) * 2 / dim)[None]
        self.cs = torch.stack([ang.cos(), ang.sin()], -1).float().contiguous().cuda()

    def step(self, e, x, pos, start, length, max_new, max_len, scratch=None, out=None, window=0):
        """x: fused rows [n][(heads + 2 kv_heads) dim]; everything enqueued on e."""
        from macseek_b200 import attn, kv8
        n = x.shape[0]
        q, k, v = (x[:, a * self.dim:b * self.dim].unflatten(1, (-1, self.dim)) for a, b in (
            (0, self.heads), (self.heads, self.heads + self.kv_heads), (self.heads + self.kv_heads, self.heads + 2 * self.kv_heads)))
        attn.encode_head_norm_rope(e, q, k, self.qw, self.kw, 1e-6, self.cs, pos, q, k, halves=True)
        batch = kv8.Batch(start, length, self.table, n, max_new, max_len)
        kv8.encode_kv8_write(e, self.cache, batch, k, v)
        out = torch.empty(n, self.heads, self.dim, dtype=x.dtype, device="cuda") if out is None else out
        kv8.encode_kv8_attn(e, self.cache, batch, q, out, kv8.attn_scratch(self.cache, batch, self.heads) if scratch is None else scratch, window=window)
        return q, out

    def check(self, q, out, seqs, window=0):
        c = R.Case.__new__(R.Case)
        c.seqs, c.kv_heads, c.dim, c.block, c.table_host = seqs, self.kv_heads, self.dim, self.block, self.table_host
        c.k, c.v, c.ks, c.vs = self.cache.k, self.cache.v, self.cache.k_scale, self.cache.v_scale
        c.start_host = [0]
        for n, _ in seqs:
            c.start_host.append(c.start_host[-1] + n)
        ref, tol = R.attn_ref(c, q, out, self.dim ** -0.5, window)
        assert ((out.double() - ref).abs() <= tol).all()


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dt,window", (("f32", 0), ("bf16", 0), ("bf16", 100)))
def test_prompts_then_tokens(dt, window):
    """Prompts of several lengths, a chunk behind one of them, then tokens one by one across the ends of blocks."""
    m = Model(8, 2, 64, 32, dt, seqs=3, blocks_each=12)
    e = enc()
    lens = [0, 0, 0]
    for new in ([200, 1, 63], [30, 17, 1], *([[1, 1, 1]] * 5), [1, 4, 2]):
        start = [0]
        for s, n in enumerate(new):
            start.append(start[-1] + n)
            lens[s] += n
        x = torch.randn(start[-1], 12 * 64, generator=m.g).to(R.DT[dt]).cuda()
        pos = i32(sum(([lens[s] - n + i for i in range(n)] for s, n in enumerate(new)), []))
        was = x.clone()
        q, out = m.step(e, x, pos, i32(start), i32(lens), max(new), max(lens), window=window)
        e.wait()
        m.check(q, out, list(zip(new, lens)), window)
        # the rows that were written are the cache's, rounded to its format: half a step of the value or of the scale's smallest
        for s, n in enumerate(new):
            for which, rows in (("k", x[:, 8 * 64:10 * 64]), ("v", was[:, 10 * 64:])):
                c = R.Case.__new__(R.Case)
                c.seqs, c.block, c.table_host = list(zip(new, lens)), 32, m.table_host
                c.k, c.v, c.ks, c.vs = m.cache.k, m.cache.v, m.cache.k_scale, m.cache.v_scale
                held = c.held(s, which, lens[s] - n).transpose(0, 1)
                want = rows[start[s]:start[s + 1]].unflatten(1, (2, 64)).double()
                assert ((held - want).abs() <= want.abs() * 2.0 ** -4 + float(c.ks.max()) * 2.0 ** -9).all()


def test_captured_steps_follow_their_arrays():
    """A captured token step replayed as the sequences grow, its lengths and positions changed between replays."""
    m = Model(16, 2, 128, 64, "bf16", seqs=4, blocks_each=8, seed=3)
    e0 = enc()
    lens = [1, 63, 64, 200]
    x = torch.randn(sum(lens), 20 * 128, generator=m.g).bfloat16().cuda()
    start = [0, 1, 64, 128, 328]
    m.step(e0, x, i32([p for n in lens for p in range(n)]), i32(start), i32(lens), 200, 200)
    e0.wait()
    x, pos, start, length = torch.zeros(4, 20 * 128, dtype=torch.bfloat16, device="cuda"), i32([0] * 4), i32([0, 1, 2, 3, 4]), i32(lens)
    from macseek_b200 import kv8
    scratch = kv8.attn_scratch(m.cache, kv8.Batch(start, length, m.table, 4, 1, 512), 16)
    out = torch.zeros(4, 16, 128, dtype=torch.bfloat16, device="cuda")
    keep = (m.cache.k.clone(), m.cache.v.clone(), m.cache.k_scale.clone(), m.cache.v_scale.clone())
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        m.step(enc(s), x, pos, start, length, 1, 512, scratch, out)      # once before, as any program does
    s.synchronize()
    for a, b in zip((m.cache.k, m.cache.v, m.cache.k_scale, m.cache.v_scale), keep):
        a.copy_(b)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        q, _ = m.step(enc(torch.cuda.current_stream()), x, pos, start, length, 1, 512, scratch, out)
    for t in range(70):
        lens = [n + 1 for n in lens]
        x.copy_(torch.randn(4, 20 * 128, generator=m.g).bfloat16())
        pos.copy_(i32([n - 1 for n in lens]))
        length.copy_(i32(lens))
        graph.replay()
        if t % 10 == 0 or t > 66:
            torch.cuda.synchronize()
            m.check(q, out, [(1, n) for n in lens])
    enc().wait()


def test_calls_on_two_streams_at_once():
    from macseek_b200 import kv8
    cases = [R.Case([(1, 3000), (2, 800)], 2, 128, 64, seed=1), R.Case([(300, 700)], 2, 64, 16, seed=2), R.Case([(1, 900)], 4, 64, 32, seed=3)]
    streams = [torch.cuda.Stream() for _ in cases]
    work = []
    for c, s in zip(cases, streams):
        q = c.randn(c.rows, c.kv_heads * 4, c.dim, dt="bf16")
        work.append((c, s, q, torch.zeros_like(q), c.cache(), c.batch()))
    scratch = [kv8.attn_scratch(w[4], w[5], w[2].shape[1]) for w in work]
    torch.cuda.synchronize()
    for _ in range(20):
        for (c, s, q, out, cache, batch), sc in zip(work, scratch):
            kv8.encode_kv8_attn(enc(s), cache, batch, q, out, sc)
    torch.cuda.synchronize()
    for c, s, q, out, *_ in work:
        check_attn(c, q, out, torch.zeros_like(out), c.dim ** -0.5, 0, None)


def test_blocks_beyond_32_bits():
    """A cache of over 4 GiB of codes: the last blocks, written, read and attended to by both kernels."""
    from macseek_b200 import kv8
    n, heads, dim, block = 70000, 8, 128, 64
    k, v = (torch.empty(n, heads, block, dim, dtype=torch.uint8, device="cuda") for _ in range(2))
    ks, vs = torch.ones(n, heads, device="cuda"), torch.ones(n, heads, device="cuda")
    assert k.numel() > 2 ** 32
    cache = kv8.Cache.of(k, v, ks, vs)
    g = torch.Generator().manual_seed(1)
    e = enc()
    c = R.Case.__new__(R.Case)
    c.kv_heads, c.dim, c.block, c.device, c.g = heads, dim, block, "cuda", g
    c.table_host = torch.tensor([[n - 1, 3, n - 2, n - 7]])
    c.k, c.v, c.ks, c.vs, c.start_host = k, v, ks, vs, [0, 200]
    table = c.table_host.int().cuda()
    rows = [c.randn(200, heads, dim, dt="bf16") for _ in range(2)]
    batch = kv8.Batch(i32([0, 200]), i32([200]), table, 200, 200, 200)
    kv8.encode_kv8_write(e, cache, batch, *rows)
    back = [torch.empty_like(r) for r in rows]
    kv8.encode_kv8_read(e, cache, batch, *back)
    e.wait()
    for a, b in zip(rows, back):
        assert ((a.double() - b.double()).abs() <= a.double().abs() * 2.0 ** -4 + 2.0 ** -15).all()
    for new in (1, 200):
        c.seqs, c.start_host = [(new, 200)], [0, new]
        batch = kv8.Batch(i32([0, new]), i32([200]), table, new, new, 200)
        q = c.randn(new, 64, dim, dt="bf16", mul=2.0)
        out = torch.zeros_like(q)
        kv8.encode_kv8_attn(e, cache, batch, q, out, kv8.attn_scratch(cache, batch, 64))
        e.wait()
        check_attn(c, q, out, out, dim ** -0.5, 0, None)
