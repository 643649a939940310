"""Attention over the 8-bit cache at the ends of what its kernels hold: keys far above the others."""
import pytest
import torch

import kv8_ref as R
from test_kv8_gpu import check_attn, enc

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", ("f32", "f16", "bf16"))
@pytest.mark.parametrize("n,dim", ((1, 64), (600, 64), (600, 128)))
def test_attention_where_one_key_is_far_above_the_others(n, dim, dt):
    """One key, or two, about 100, 400, 600 or 5000 binary exponents above all before it, at each of 16 places of a tile that is not the first."""
    from macseek_b200 import kv8
    G, scale = 8, 2.0 ** -8
    c = R.Case([(n, 1000)], 4, dim, 16, seed=3)
    c.k.fill_(0)
    c.ks.fill_(1)
    blk = int(c.table_host[0, 20])
    q = torch.zeros(c.rows, 4 * G, dim, dtype=R.DT[dt], device="cuda")
    q[:, :, 5] = torch.tensor([100.0, 400.0, 600.0, 5000.0], device="cuda").repeat(8).to(R.DT[dt]) * 0.6875      # times ln 2, about
    cache, batch, e = c.cache(), c.batch(), enc()
    scratch = kv8.attn_scratch(cache, batch, 4 * G)
    for places in [(p,) for p in range(16)] + [(6, 7), (14, 15), (0, 6)]:
        c.k[blk] = 0
        for p in places:
            c.k[blk, :, p, 5] = 0x78                                 # 256
        out = torch.zeros_like(q)
        kv8.encode_kv8_attn(e, cache, batch, q, out, scratch, scale=scale)
        e.wait()
        check_attn(c, q, out, torch.zeros_like(out), scale, 0, None)


@pytest.mark.parametrize("dt", ("f32", "f16", "bf16"))
def test_rows_that_see_no_block_are_zero_beside_rows_that_do(dt):
    """The first blocks of a prompt are not there: its first rows see nothing, whatever scale the later blocks' values have."""
    from macseek_b200 import _lib, kv8
    n, dim, gone = 1100, 64, 144              # (a tile of 256 rows is 32 tokens: 16 of them see nothing)
    c = R.Case([(n, n)], 4, dim, 16, seed=8)
    c.table[0, :gone // 16] = -1
    cache, batch, e = c.cache(), c.batch(), enc()
    for ex in (0, 5, 6, -20) if dt == "f16" else (0, 6, 14, 24, -30):
        c.vs.fill_(2.0 ** ex)
        q = c.randn(n, 32, dim, dt=dt, mul=0.1)
        out = torch.full_like(q, 7)
        kv8.encode_kv8_attn(e, cache, batch, q, out, kv8.attn_scratch(cache, batch, 32))
        torch.cuda.synchronize()
        assert _lib.device_status() == 4
        assert (out[:gone] == 0).all()
        k, v = c.held(0, "k", gone), c.held(0, "v", gone)
        seen = torch.arange(gone, n, device="cuda")[None] <= torch.arange(gone, n, device="cuda")[:, None]
        for h in (0, 13, 31):
            w = torch.softmax((q[gone:, h].double() @ k[h // 8].T * dim ** -0.5).masked_fill(~seen, -torch.inf), 1)
            # weights and the output rounded to 11 bits (bf16: the output to 8), all else far finer
            assert ((w @ v[h // 8]) - out[gone:, h].double()).abs().max() <= v.abs().max() * (2.0 ** -11 + 2.0 ** -14 + R.half_step(R.DT[dt])[0])


def one_long_context(S, n, L, dt, kv=8, G=8, dim=128, block=64):
    """S sequences of n new tokens over one context of L tokens that they share: keys 0 but for the first, values of one sign."""
    from macseek_b200 import kv8
    g = torch.Generator().manual_seed(3)
    nb = -(-L // block)
    cache = kv8.Cache(nb, kv, dim, block)
    cache.v.copy_((torch.rand(cache.v.shape, generator=g) * 128 + 128).to(R.FP8).view(torch.uint8))
    cache.v_scale.fill_(2.0 ** -8)
    i32 = dict(dtype=torch.int32, device="cuda")
    batch = kv8.Batch(torch.arange(S + 1, **i32) * n, torch.full((S,), L, **i32), torch.arange(nb, **i32)[None].expand(S, -1).contiguous(), S * n, n, L)
    cache.k[0, :, 0, 0], cache.v[0, :, 0] = 0x38, 0x58               # 1, 16
    v = (R.values(cache.v) * 2.0 ** -8).transpose(0, 1).reshape(kv, -1, dim)[:, :L]
    q = torch.zeros(S * n, kv * G, dim, dtype=R.DT[dt], device="cuda")
    q[:, :, 0] = 1
    return cache, batch, q, v


@pytest.mark.parametrize("dt", ("f32", "f16", "bf16"))
@pytest.mark.parametrize("S,n", ((128, 1), (1, 512)))
@pytest.mark.parametrize("gap", (12.0, 15.0, 16.0, 17.5))
def test_attention_keeps_small_weights_beside_a_large_one(S, n, dt, gap):
    """The first key's logit is `gap` above those of thousands of others, whose weights together are a share of the sum that the output shows.

    All values have one sign, so that weights off by 2^-11 (F32: 2^-21) and 2^x by 2^-20, the largest's among them, count by the result; a logit is
    off by gap 2^-21, which counts by the share; sums over L tokens, 16 at a time and F32 in two halves, are off by (L / 8 + 32) 2^-23 of themselves."""
    from macseek_b200 import kv8
    L = 8192
    cache, batch, q, v = one_long_context(S, n, L, dt)
    out, e = torch.zeros_like(q), enc()
    kv8.encode_kv8_attn(e, cache, batch, q, out, kv8.attn_scratch(cache, batch, 64), scale=gap)
    e.wait()
    pos = torch.arange(L - n, L, device="cuda")
    small = float(torch.exp(torch.tensor(-gap, dtype=torch.float64)))
    total = 1 + small * pos.double()[:, None]
    half, tiny = R.half_step(q.dtype)
    share = (total - 1) / total
    weight = (2.0 ** -21 if dt == "f32" else 2.0 ** -11) + 2.0 ** -20
    for h in range(64):
        rest = v[h // 8, 1:].cumsum(0)[pos - 1]
        ref = (v[h // 8, 0] + small * rest) / total                  # [n][dim]
        tol = (weight + (L / 8 + 32) * 2.0 ** -23) * ref + share * gap * 2.0 ** -21
        got = out.view(S, n, 64, 128)[:, :, h].double()
        assert ((got - ref).abs() <= tol * (1 + half) + half * ref.abs() + tiny).all(), (h, float((got - ref).abs().max()), float(tol.max()))


@pytest.mark.parametrize("S,n", ((128, 1), (1, 512)))
def test_attention_sums_of_f32_rows_keep_what_is_below_their_last_bit(S, n):
    """Tens of thousands of weights, each of them below the last bit of the first key's, that together are not.

    As above; but sums are begun anew after 1024 keys at most (few rows: 512 of a warp's), and what each held is added in 32 bits."""
    from macseek_b200 import kv8
    L, gap = 40000, 20.0
    cache, batch, q, v = one_long_context(S, n, L, "f32")
    out, e = torch.zeros_like(q), enc()
    kv8.encode_kv8_attn(e, cache, batch, q, out, kv8.attn_scratch(cache, batch, 64), scale=gap)
    e.wait()
    pos = torch.arange(L - n, L, device="cuda")
    small = float(torch.exp(torch.tensor(-gap, dtype=torch.float64)))
    total = 1 + small * pos.double()[:, None]
    adds = L / 1024 if n > 1 else L / 4 / 512                        # (a warp of a block of few rows has a quarter of a part's keys)
    for h in range(0, 64, 7):
        ref = (v[h // 8, 0] + small * v[h // 8, 1:].cumsum(0)[pos - 1]) / total
        tol = (2.0 ** -21 + 2.0 ** -20 + (1024 / 8 + 32) * 2.0 ** -23 + adds * 2.0 ** -24) * ref + (total - 1) / total * gap * 2.0 ** -21
        assert ((out.view(S, n, 64, 128)[:, :, h].double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("dt", ("f32", "f16", "bf16"))
@pytest.mark.parametrize("S,n,kv,dim,L", ((128, 1, 8, 128, 200000), (1, 512, 8, 128, 200000), (1, 256, 1, 64, 400000)))
def test_attention_of_long_contexts_is_not_biased(S, n, kv, dim, L, dt):
    """Values of one sign under random weights: what sums cut off would make every output smaller.  (One part, several, and parts of many rows whose
    sums are begun anew.)

    Roundings of weights and outputs cancel in the mean (two heads, 64 rows, their dims: their mean is below 2^-11 / 60); what does not is 2^-23 of
    a sum at every 16 keys, for 1024 keys of F32 rows and 16384 of others, and 2^-18 of a weight."""
    from macseek_b200 import kv8
    sc, G = dim ** -0.5, 8
    cache, batch, q, v = one_long_context(S, n, L, dt, kv=kv, dim=dim)
    g = torch.Generator(device="cuda").manual_seed(5)
    cache.k.copy_(torch.randn(cache.k.shape, generator=g, device="cuda").to(R.FP8).view(torch.uint8))
    q.copy_(torch.randn(q.shape, generator=g, device="cuda"))
    out, e = torch.zeros_like(q), enc()
    scratch = kv8.attn_scratch(cache, batch, kv * G)
    scratch.fill_(255)                                               # NaN
    kv8.encode_kv8_attn(e, cache, batch, q, out, scratch, scale=sc)
    e.wait()
    err = []
    for h in (3, kv * G - 4):
        k = R.values(cache.k)[:, h // G].reshape(-1, dim)[:L]
        rows = torch.arange(S * n - 64, S * n, device="cuda")
        lg = (q[rows, h].double() @ k.T * sc).masked_fill(torch.arange(L, device="cuda")[None] > (L - n + rows % n)[:, None], -torch.inf)
        ref = torch.softmax(lg, 1) @ v[h // G]
        err.append((out[rows, h].double() / ref - 1).mean())
    keys = 1024 if dt == "f32" else 16384
    bias = abs(float(torch.stack(err).mean()))
    assert bias <= keys / 16 * 2.0 ** -23 + 2.0 ** -18 + (0 if dt == "f32" else R.half_step(R.DT[dt])[0] / 60), bias


def broken_starts(c):
    """(start's entries to change, the sequences that are right then)."""
    n = len(c.seqs)
    yield {2: c.rows + 70}, [s for s in range(n) if s not in (1, 2)]
    yield {2: 10 ** 6}, [s for s in range(n) if s not in (1, 2)]
    yield {1: -3, n - 1: 2 ** 31 - 1}, [s for s in range(n) if s not in (0, 1, n - 2, n - 1)]
    yield {3: 0}, [s for s in range(n) if s not in (2, 3)]             # (sequence 3 would have more rows than any may)


@pytest.mark.parametrize("seqs,G", (([(5, 2000 + 7 * i) for i in range(7)], 8), ([(1, 900), (3, 700), (2, 1000), (1, 50), (4, 800)], 2), ([(80, 3000)] * 5, 8)))
def test_broken_starts_leave_the_other_sequences_right_in_several_parts(seqs, G):
    """A start that falls or lies outside hides no sequence behind it from the kernel that joins parts."""
    from macseek_b200 import _lib, kv8
    c = R.Case(seqs, 2, 64, 16, seed=11, pad=3)
    e, q = enc(), c.randn(c.rows, 2 * G, 64)
    outs = []
    start = c.start.clone()
    for change, good in [({}, range(len(seqs)))] + list(broken_starts(c)):
        c.start.copy_(start)
        for i, x in change.items():
            c.start[i] = x
        cache, batch = c.cache(), c.batch()
        out = torch.full_like(q, 7)
        scratch = kv8.attn_scratch(cache, batch, 2 * G)
        scratch.fill_(255)
        kv8.encode_kv8_attn(e, cache, batch, q, out, scratch)
        torch.cuda.synchronize()
        assert _lib.device_status() == (4 if change else 0)
        if not change:
            check_attn(c, q, out, torch.full_like(q, 7), 0.125, 0, None)
        outs.append(out)
        for s in good:
            r = slice(c.start_host[s], c.start_host[s] + seqs[s][0])
            assert torch.equal(out[r], outs[0][r]), (change, s)
        assert (out[c.start_host[-1]:] == 7).all()


RAGGED = [[(300, 300), (5, 50), (40, 40), (33, 70), (1, 9), (64, 64), (2, 30), (17, 200)], [(700, 900), (1, 1), (3, 64), (0, 20), (2, 65), (9, 9)]]


@pytest.mark.parametrize("seqs", RAGGED)
@pytest.mark.parametrize("block,dt", ((16, "f32"), (64, "bf16"), (128, "f16"), (32, "bf16")))
def test_broken_starts_leave_the_other_sequences_right_in_ragged_writes_and_reads(seqs, block, dt):
    from macseek_b200 import _lib, kv8
    e = enc()

    def make():
        return R.Case(seqs, 3, 64, block, seed=12, pad=3)
    c = make()
    k, v = c.randn(c.rows, 3, 64, dt=dt), c.randn(c.rows, 3, 64, dt=dt)
    kv8.encode_kv8_write(e, c.cache(), c.batch(), k, v)
    whole = c
    rows = [torch.full_like(k, 7), torch.full_like(k, 7)]
    kv8.encode_kv8_read(e, c.cache(), c.batch(), *rows)
    e.wait()
    for change, good in broken_starts(c):
        c, fresh = make(), make()
        for i, x in change.items():
            c.start[i] = x
        good = [s for s in good if seqs[s][0]]
        kv8.encode_kv8_write(e, c.cache(), c.batch(), k, v)
        torch.cuda.synchronize()
        assert _lib.device_status() == 4
        mine = torch.zeros(c.k.shape[0], dtype=torch.bool)
        for s, (n, l) in enumerate(seqs):
            if s in good:
                mine[c.table_host[s, :-(-l // block)]] = True
        mine = mine.cuda()
        for a, b, f in ((c.k, whole.k, fresh.k), (c.v, whole.v, fresh.v), (c.ks, whole.ks, fresh.ks), (c.vs, whole.vs, fresh.vs)):
            assert torch.equal(a[mine].nan_to_num(-1) if a.is_floating_point() else a[mine], b[mine].nan_to_num(-1) if b.is_floating_point() else b[mine])
            assert torch.equal(a[~mine].nan_to_num(-1) if a.is_floating_point() else a[~mine], f[~mine].nan_to_num(-1) if f.is_floating_point() else f[~mine])
        ko, vo = torch.full_like(k, 7), torch.full_like(k, 7)
        whole.start.copy_(c.start)
        kv8.encode_kv8_read(e, whole.cache(), whole.batch(), ko, vo)
        torch.cuda.synchronize()
        assert _lib.device_status() == 4
        keep = torch.zeros(c.rows, dtype=torch.bool)
        for s in good:
            keep[c.start_host[s]:c.start_host[s] + seqs[s][0]] = True
        keep = keep.cuda()
        for got, want in ((ko, rows[0]), (vo, rows[1])):
            assert torch.equal(got[keep], want[keep]) and (got[~keep] == 7).all()


@pytest.mark.parametrize("dt", ("f32", "bf16"))
@pytest.mark.parametrize("seqs,heads,G,window", (([(1, 1000), (3, 500), (1, 90)], 2, 8, 77), ([(1, 4000)], 8, 8, 1500), ([(90, 700), (200, 900)], 4, 8, 100),
                                                 ([(600, 2000)], 4, 8, 1000), ([(64, 300)], 1, 16, 1)))
def test_blocks_before_the_window_need_not_be_there(seqs, heads, G, window, dt):
    """A program with a sliding window gives blocks back that no row sees any more; their ids in the table are anything then."""
    from macseek_b200 import kv8
    for dim in (64, 128):
        c = R.Case(seqs, heads, dim, 16, seed=13, pad=1)
        for s, (n, l) in enumerate(seqs):
            gone = max(0, l - n - window + 1) // 16
            c.table[s, :gone] = torch.tensor([-1, 2 ** 31 - 1, c.k.shape[0]], dtype=torch.int32, device="cuda").repeat(gone)[:gone]
        cache, batch, e = c.cache(), c.batch(), enc()
        q = c.randn(c.rows, heads * G, dim, dt=dt, mul=3.0)
        out = torch.full_like(q, 7)
        kv8.encode_kv8_attn(e, cache, batch, q, out, kv8.attn_scratch(cache, batch, heads * G), window=window)
        e.wait()                                                     # raises where the batch is called broken
        check_attn(c, q, out, torch.full_like(q, 7), dim ** -0.5, window, None)


@pytest.mark.parametrize("dt", ("f32", "bf16"))
@pytest.mark.parametrize("n", (1, 600, 1000))
def test_attention_of_tiny_queries_under_a_large_scale(n, dt):
    """Queries near the smallest numbers and a scale that makes ordinary logits of them."""
    from macseek_b200 import kv8
    c = R.Case([(n, 1100)], 4, 64, 16, seed=15)
    cache, batch, e = c.cache(), c.batch(), enc()
    base = c.randn(c.rows, 32, 64, dt=dt)
    for ex in (40, 60, 70, 90, 110):
        q = base * 2.0 ** -ex
        out = torch.zeros_like(q)
        kv8.encode_kv8_attn(e, cache, batch, q, out, kv8.attn_scratch(cache, batch, 32), scale=2.0 ** (ex - 3))
        e.wait()
        check_attn(c, q, out, torch.zeros_like(out), 2.0 ** (ex - 3), 0, None)


@pytest.mark.parametrize("dt", ("f32", "f16", "bf16"))
@pytest.mark.parametrize("n", (1, 600, 1000))
@pytest.mark.parametrize("sign", (1.0, -1.0))
def test_attention_over_logits_beyond_the_steps_of_32_bits(n, dt, sign):
    """Logits of 2^20 to 2^60, whose last bits are larger than an exponent: the largest key's value is the result, wherever it lies."""
    from macseek_b200 import kv8
    G, dim = 8, 64
    c = R.Case([(n, 1100)], 4, dim, 16, seed=14)
    c.ks.fill_(1)
    cache, batch, e = c.cache(), c.batch(), enc()
    scratch = kv8.attn_scratch(cache, batch, 4 * G)
    q = torch.zeros(c.rows, 4 * G, dim, dtype=R.DT[dt], device="cuda")
    q[:, :, 3] = torch.linspace(1, 1.9375, 16, device="cuda").repeat(2).to(q.dtype)
    for ex in (20, 24, 26, 27, 28, 29, 30, 31, 32, 34, 36, 40, 60):
        for at in (5, 70, 333):
            c.k.fill_(0)
            c.k[:, :, :, 3] = 0x70 if sign > 0 else 0x78             # 128, 256
            c.k[c.table_host[0, at // 16], :, at % 16, 3] = 0x78 if sign > 0 else 0x70
            out = torch.zeros_like(q)
            kv8.encode_kv8_attn(e, cache, batch, q, out, scratch, scale=sign * 2.0 ** (ex - 8))
            e.wait()
            v = c.held(0, "v")[:, at].repeat_interleave(G, 0)
            sees = torch.arange(1100 - n, 1100, device="cuda")[:, None, None] >= at
            bad = sees & ((out.double() - v[None]).abs() > v.abs() * (2.0 ** -11 + 2.0 ** -20 + R.half_step(q.dtype)[0]) + 2.0 ** -30)
            assert not (bad | out.isnan()).any(), (ex, at, int(bad.sum()), out.isnan().sum())


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("dim", (64, 128))
def test_attention_whose_sums_begin_anew_under_peaked_weights(seed, dim):
    """F32 rows over a little more than 1024 keys, a few of which have nearly all the weight: what O held is taken when all of it is there."""
    from macseek_b200 import kv8
    seqs = [(151, 151), (24, 50), (191, 897 + 300 * (seed % 2)), (200, 1107), (77, 77), (271, 2580)]
    c = R.Case(seqs, 3, dim, 16, seed=seed, pad=1)
    cache, batch, e = c.cache(), c.batch(), enc()
    q = c.randn(c.rows, 6, dim, mul=10.0 if seed < 3 else 3.0)
    sinks = c.randn(6, mul=3.0)
    scratch = kv8.attn_scratch(cache, batch, 6)
    for _ in range(3):
        out = torch.full_like(q, 7)
        kv8.encode_kv8_attn(e, cache, batch, q, out, scratch, sinks=sinks)
        e.wait()
        check_attn(c, q, out, torch.full_like(q, 7), dim ** -0.5, 0, sinks)
