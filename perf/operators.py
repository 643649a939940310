"""Operators of grouped-query attention over an 8-bit cache: cases, inputs, plain forms and definitions in 64 bits.

    norm_rope   RMSNorm of every query and key head with the position rotation in the same pass
    write       new key / value rows quantised into a paged e4m3 cache, one power-of-two scale per block of tokens and head
    read        rows of that cache as F32 / F16 / BF16
    attn        attention of the newest query rows of each sequence over the cache

A cache is codes [blocks][heads][block][dim] (e4m3, as bytes) and scales [blocks][heads] for keys and for values.  A batch of
sequences is seq_start [n+1] (rows of the new tokens), kv_len [n] (tokens with the new ones) and table [n][..] (block ids); rows
behind seq_start[n] are padding and stay as they are."""
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6
FP8 = torch.float8_e4m3fn
MIN_EXP, MAX_EXP = -50, 50      # exponents of scales: a block of zeros has the smallest, values beyond 448 times the largest become that


def listed():
    return [
        # one token of the decode step behind the query / key projections, rotation on the last 64 dims (pairs), 200K positions
        dict(name="norm_rope_token", op="norm_rope", tokens=1, q_heads=64, kv_heads=8, dim=128, rot=64, first=64, halves=False, type="f32", positions=200000),
        # a prompt of 4096 tokens, whole heads rotated by halves
        dict(name="norm_rope_prompt", op="norm_rope", tokens=4096, q_heads=64, kv_heads=8, dim=128, rot=128, first=0, halves=True, type="bf16", positions=65536),
        # an odd chunk with small heads of which a half is rotated
        dict(name="norm_rope_chunk", op="norm_rope", tokens=999, q_heads=32, kv_heads=4, dim=64, rot=32, first=0, halves=True, type="f16", positions=65536),
        # one new token for each of 64 sequences: older rows of the last block may have to move to a larger scale
        dict(name="write_tokens", op="write", seqs=64, new=1, ctx=999, ragged=True, kv_heads=8, dim=128, block=64, type="f32"),
        # prompts of several lengths, some behind a cached prefix
        dict(name="write_prompts", op="write", seqs=4, new=4096, ctx=999, ragged=True, kv_heads=8, dim=128, block=64, type="bf16"),
        # a short prefix read back
        dict(name="read_chunk", op="read", seqs=1, new=999, ctx=17, ragged=False, kv_heads=4, dim=64, block=16, type="f16"),
        # the caches of 16 sequences read back
        dict(name="read_prompts", op="read", seqs=16, new=8192, ctx=0, ragged=True, kv_heads=8, dim=128, block=64, type="bf16"),
        # one token of one short sequence: latency
        dict(name="attn_token", op="attn", seqs=1, new=1, ctx=998, ragged=False, q_heads=64, kv_heads=8, dim=128, block=64, window=0, sinks=False, type="f32"),
        # one token for each of 64 sequences of ragged lengths
        dict(name="attn_tokens", op="attn", seqs=64, new=1, ctx=8191, ragged=True, q_heads=64, kv_heads=8, dim=128, block=64, window=0, sinks=False, type="bf16"),
        # one token behind 200K others
        dict(name="attn_token_far", op="attn", seqs=1, new=1, ctx=199999, ragged=False, q_heads=64, kv_heads=8, dim=128, block=64, window=0, sinks=False, type="bf16"),
        # a whole prompt
        dict(name="attn_prompt", op="attn", seqs=1, new=4096, ctx=0, ragged=False, q_heads=64, kv_heads=8, dim=128, block=64, window=0, sinks=False, type="bf16"),
        # chunks of ragged prompts behind ragged contexts, small heads, sinks and a sliding window
        dict(name="attn_chunks", op="attn", seqs=5, new=333, ctx=8192, ragged=True, q_heads=32, kv_heads=4, dim=64, block=16, window=4096, sinks=True, type="f16"),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["norm_rope", "write", "read", "attn", "attn", "attn"])
    kind = rng.choice(sorted(TYPES))
    dim, kv_heads, group = rng.choice([64, 128]), rng.choice([1, 2, 3, 4, 5, 8]), rng.choice([1, 2, 3, 4, 6, 7, 8])
    if op == "norm_rope":
        rot = rng.choice([32, 64, dim])
        return dict(op=op, tokens=_spread(rng, 1, 4096), q_heads=kv_heads * group, kv_heads=kv_heads, dim=dim, rot=rot,
                    first=rng.choice([0, dim - rot]), halves=rng.random() < 0.5, type=kind, positions=rng.choice([8192, 65536]))
    c = dict(op=op, kv_heads=kv_heads, dim=dim, block=rng.choice([16, 32, 64, 128]), ragged=rng.random() < 0.7, type=kind)
    if op != "attn":
        c["seqs"] = _spread(rng, 1, 64)
        c["new"] = rng.choice([1, _spread(rng, 1, max(1, min(4096, 16384 // c["seqs"])))])
        c["ctx"] = rng.choice([0, _spread(rng, 1, 999)])
        return c
    c.update(q_heads=kv_heads * group, window=rng.choice([0, 0, 0, _spread(rng, 16, 4096)]), sinks=rng.random() < 0.3)
    if rng.random() < 0.5:                                      # single tokens and short drafts
        c["seqs"], c["new"] = _spread(rng, 1, 64), rng.choice([1, 1, 1, 2, 4, 5])
        c["ctx"] = _spread(rng, 1, min(131072, 64 * 4096 // (c["seqs"] * c["new"])))
    else:                                                       # chunks and prompts
        c["seqs"], c["new"] = _spread(rng, 1, 6), _spread(rng, 17, 2048)
        c["ctx"] = rng.choice([0, _spread(rng, 1, 2048)])
        while c["seqs"] > 1 and c["seqs"] * c["new"] * c["q_heads"] * dim * (c["new"] + 2 * c["ctx"]) > 4096 * 4096 * 64 * 128:
            c["seqs"] -= 1
    return c


# ------------------------------------------------------------------------------------------------ inputs
def _lengths(case, seed):
    """(new, ctx) of every sequence: the same ones for every seed, in another order; the longest are what the case says."""
    n = case["seqs"]
    if not case["ragged"]:
        return [case["new"]] * n, [case["ctx"]] * n
    g = torch.Generator().manual_seed(case["new"] * 7919 + case["ctx"])
    new = torch.randint(1, case["new"] + 1, (n,), generator=g)
    ctx = torch.randint(0, case["ctx"] + 1, (n,), generator=g)
    new[int(torch.randint(0, n, (1,), generator=g))] = case["new"]
    ctx[int(torch.randint(0, n, (1,), generator=g))] = case["ctx"]
    order = torch.randperm(n, generator=torch.Generator().manual_seed(seed))
    return new[order].tolist(), ctx[order].tolist()


def _batch(case, seed, g, dev):
    new, ctx = _lengths(case, seed)
    start = [0]
    for v in new:
        start.append(start[-1] + v)
    length = [a + b for a, b in zip(new, ctx)]
    per = -(-max(length) // case["block"])
    blocks = case["seqs"] * per + 1
    table = (torch.randperm(blocks - 1, device=dev, generator=g).to(torch.int32) + 1)[:case["seqs"] * per]
    rows = start[-1] + (5 if case["ragged"] else 0)             # a padded batch
    i32 = dict(dtype=torch.int32, device=dev)
    return dict(seq_start=torch.tensor(start, **i32), kv_len=torch.tensor(length, **i32),
                table=table.reshape(case["seqs"], per).contiguous(), rows=rows, blocks=blocks,
                max_new=max(new), max_len=max(length))


def _codes(shape, g, dev):
    """Codes of normal values whose largest of a block lies near the end of the format."""
    out = torch.empty(shape, dtype=torch.uint8, device=dev)
    flat = out.view(-1)
    for i in range(0, flat.numel(), 1 << 28):
        part = flat[i:i + (1 << 28)]
        part.copy_(torch.randn(part.numel(), device=dev, generator=g).mul_(112).clamp_(-448, 448).to(FP8).view(torch.uint8))
    return out


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt, D, Hk = TYPES[case["type"]], case["dim"], case["kv_heads"]
    rand = lambda *s: torch.randn(*s, device=dev, generator=g)  # noqa: E731
    s = dict(case)
    if case["op"] == "norm_rope":
        T, Hq, half = case["tokens"], case["q_heads"], case["rot"] // 2
        x = rand(T, (Hq + 2 * Hk) * D).to(dt)                   # the fused projection's rows: queries, keys, values
        ang = torch.arange(case["positions"], device=dev, dtype=torch.float64)[:, None] \
            * torch.pow(10000.0, -torch.arange(half, device=dev, dtype=torch.float64) / half)
        first = int(torch.randint(0, max(1, case["positions"] - T), (1,), device=dev, generator=g))
        s.update(q=x[:, :Hq * D].unflatten(1, (Hq, D)), k=x[:, Hq * D:(Hq + Hk) * D].unflatten(1, (Hk, D)),
                 q_w=1 + 0.2 * rand(D), k_w=1 + 0.2 * rand(D), cs=torch.stack([ang.cos(), ang.sin()], -1).float(),
                 pos=torch.arange(first, first + T, device=dev, dtype=torch.int32) % case["positions"],
                 q_out=torch.zeros(T, Hq, D, dtype=dt, device=dev), k_out=torch.zeros(T, Hk, D, dtype=dt, device=dev))
        return s
    b = _batch(case, seed, g, dev)
    shape = (b["blocks"], Hk, case["block"], D)
    scale = lambda: torch.exp2(torch.randint(-8, -5, shape[:2], device=dev, generator=g).float())  # noqa: E731
    s.update(b, k_codes=_codes(shape, g, dev), v_codes=_codes(shape, g, dev), k_scale=scale(), v_scale=scale())
    if case["op"] == "write":
        x = rand(b["rows"], 2 * Hk * D).to(dt)
        s.update(k=x[:, :Hk * D].unflatten(1, (Hk, D)), v=x[:, Hk * D:].unflatten(1, (Hk, D)))
    elif case["op"] == "read":
        s.update(k_out=torch.zeros(b["rows"], Hk, D, dtype=dt, device=dev), v_out=torch.zeros(b["rows"], Hk, D, dtype=dt, device=dev))
    else:
        Hq = case["q_heads"]
        s.update(q=(2 * rand(b["rows"], Hq, D)).to(dt), out=torch.zeros(b["rows"], Hq, D, dtype=dt, device=dev),
                 sink=rand(Hq) if case["sinks"] else None)
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    return _own(s) if own else {"norm_rope": _norm_rope, "write": _write, "read": _read, "attn": _attn}[s["op"]](s)


def _own(s):
    from macseek_b200 import attn, kv8
    from macseek_b200.core import Enc
    e = Enc()
    if s["op"] == "norm_rope":
        attn.encode_head_norm_rope(e, s["q"], s["k"], s["q_w"], s["k_w"], EPS, s["cs"], s["pos"], s["q_out"], s["k_out"],
                                   rot_first=s["first"], halves=s["halves"])
        return {"q": s["q_out"], "k": s["k_out"]}
    if "handle" not in s:                                       # what a program keeps: the cache, the batch, the scratch
        cache = kv8.Cache.of(s["k_codes"], s["v_codes"], s["k_scale"], s["v_scale"])
        batch = kv8.Batch(s["seq_start"], s["kv_len"], s["table"], s["rows"], s["max_new"], s["max_len"])
        s["handle"] = cache, batch, kv8.attn_scratch(cache, batch, s["q_heads"]) if s["op"] == "attn" else None
    cache, batch, scratch = s["handle"]
    if s["op"] == "write":
        kv8.encode_kv8_write(e, cache, batch, s["k"], s["v"])
        return _state(s)
    if s["op"] == "read":
        kv8.encode_kv8_read(e, cache, batch, s["k_out"], s["v_out"])
        return {"k": s["k_out"], "v": s["v_out"]}
    kv8.encode_kv8_attn(e, cache, batch, s["q"], s["out"], scratch, window=s["window"], sinks=s["sink"])
    return s["out"]


def _state(s):
    return {"k": s["k_codes"].view(FP8), "v": s["v_codes"].view(FP8), "k_scale": s["k_scale"], "v_scale": s["v_scale"]}


def _norm_rope(s):
    cs = s["cs"][s["pos"].long()]                               # [T][rot/2][2]
    c, n = cs[:, None, :, 0], cs[:, None, :, 1]
    out = []
    for x, w, y in ((s["q"], s["q_w"], s["q_out"]), (s["k"], s["k_w"], s["k_out"])):
        x = x.float()
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w
        part = x[..., s["first"]:s["first"] + s["rot"]]
        if s["halves"]:
            a, b = part.chunk(2, -1)
            part = torch.cat([a * c - b * n, a * n + b * c], -1)
        else:
            a, b = part[..., 0::2], part[..., 1::2]
            part = torch.stack([a * c - b * n, a * n + b * c], -1).flatten(-2)
        out.append(torch.cat([x[..., :s["first"]], part, x[..., s["first"] + s["rot"]:]], -1).to(y.dtype))
    return {"q": out[0], "k": out[1]}


def _padded(s):
    """[seqs][max_new]: row of every new token, its position, and whether there is one (others: the row behind the last)."""
    i = torch.arange(s["max_new"], device=s["kv_len"].device)
    n = (s["seq_start"][1:] - s["seq_start"][:-1])[:, None].long()
    there = i < n
    return torch.where(there, s["seq_start"][:-1, None] + i, s["rows"]), s["kv_len"][:, None] - n + i, there


def _write(s):
    BT, dev = s["block"], s["kv_len"].device
    start = (s["kv_len"] - (s["seq_start"][1:] - s["seq_start"][:-1])).long()            # position of the first new token
    touched = (s["max_new"] + 2 * BT - 2) // BT
    blk = start[:, None] // BT + torch.arange(touched, device=dev)                       # [seqs][touched]
    p = blk[..., None] * BT + torch.arange(BT, device=dev)                               # [seqs][touched][BT]
    new = (p >= start[:, None, None]) & (p < s["kv_len"][:, None, None])
    there = new.any(-1)
    ids = s["table"].gather(1, blk.clamp(max=s["table"].shape[1] - 1)).long()
    ids = torch.where(there, ids, s["blocks"])                                           # the others: a block behind the last
    row = torch.where(new, s["seq_start"][:-1, None, None] + p - start[:, None, None], 0)
    old = (p < start[:, None, None]) & there[..., None]
    any_old = old.any(-1)[..., None]                                                     # [seqs][touched][1]
    out = []
    for x, codes, scale in ((s["k"], s["k_codes"], s["k_scale"]), (s["v"], s["v_codes"], s["v_scale"])):
        v = x[row].float().permute(0, 1, 3, 2, 4)                                        # [seqs][touched][heads][BT][dim]
        m = new[:, :, None, :, None]
        amax = torch.where(m, v.abs(), 0).amax((-1, -2))
        frac, exp = torch.frexp(amax)
        exp = torch.where(amax > 0, exp - torch.where(frac <= 0.875, 9, 8), MIN_EXP).clamp(MIN_EXP, MAX_EXP)
        codes, scale = (torch.cat([t, t[:1]]) for t in (codes, scale))
        had = torch.frexp(scale[ids])[1] - 1
        exp = torch.where(any_old, torch.maximum(exp, had), exp)
        was = codes[ids]
        moved = torch.ldexp(was.view(FP8).float(), (had - exp)[..., None, None])
        put = torch.where(m, torch.ldexp(v, -exp[..., None, None]).clamp(-448, 448), moved).to(FP8).view(torch.uint8)
        codes[ids] = torch.where(m | old[:, :, None, :, None], put, was)
        scale[ids] = torch.ldexp(torch.ones_like(amax), exp)
        out += [codes[:-1].view(FP8), scale[:-1]]
    return dict(zip(("k", "k_scale", "v", "v_scale"), out))


def _rows_of(s, codes, scale, pos, seq):
    """Values at positions `pos` of sequences `seq` (same shapes): [..., heads, dim]."""
    pos = pos.clamp(0, s["table"].shape[1] * s["block"] - 1).long()
    ids = s["table"][seq, pos // s["block"]].long()
    return codes[ids, :, pos % s["block"]].view(FP8).float() * scale[ids][..., None]


def _read(s):
    row, pos, _ = _padded(s)
    seq = torch.arange(s["seqs"], device=row.device)[:, None].expand_as(pos)
    out = []
    for codes, scale, y in ((s["k_codes"], s["k_scale"], s["k_out"]), (s["v_codes"], s["v_scale"], s["v_out"])):
        y = torch.cat([y, y[:1]])
        y[row] = _rows_of(s, codes, scale, pos, seq).to(y.dtype)
        out.append(y[:-1])
    return {"k": out[0], "v": out[1]}


def _attn(s):
    row, qpos, there = _padded(s)
    S, N, L, D, Hk = s["seqs"], s["max_new"], s["max_len"], s["dim"], s["kv_heads"]
    G = s["q_heads"] // Hk
    dev = row.device
    kpos = torch.arange(L, device=dev).expand(S, L)
    seq = torch.arange(S, device=dev)[:, None].expand(S, L)
    held = (kpos < s["kv_len"][:, None])[..., None, None]
    k = torch.where(held, _rows_of(s, s["k_codes"], s["k_scale"], kpos, seq), 0).permute(0, 2, 3, 1)       # [S][Hk][D][L]
    q = torch.cat([s["q"], s["q"][:1]])[row].float().reshape(S, N, Hk, G, D).permute(0, 2, 1, 3, 4).reshape(S, Hk, N * G, D)
    logit = (torch.matmul(q, k) * D ** -0.5).reshape(S, Hk, N, G, L)
    k = q = None
    kp, qp = kpos[:, None, :], qpos[:, :, None]
    seen = there[:, :, None] & (kp <= qp) & (kp < s["kv_len"][:, None, None])
    if s["window"]:
        seen = seen & (kp > qp - s["window"])
    logit = logit.masked_fill_(~seen[:, None, :, None, :], -torch.inf)
    top = logit.amax(-1, keepdim=True)
    if s["sink"] is not None:
        sink = s["sink"].reshape(1, Hk, 1, G, 1)
        top = torch.maximum(top, sink)
    top = torch.where(top == -torch.inf, 0, top)
    p = logit.sub_(top).exp_()
    den = p.sum(-1, keepdim=True)
    if s["sink"] is not None:
        den = den + torch.exp(sink - top)
    v = torch.where(held, _rows_of(s, s["v_codes"], s["v_scale"], kpos, seq), 0).permute(0, 2, 1, 3)       # [S][Hk][L][D]
    o = torch.matmul(p.reshape(S, Hk, N * G, L), v).reshape(S, Hk, N, G, D) / torch.where(den > 0, den, 1)
    out = torch.cat([s["out"], s["out"][:1]])
    out[row] = o.permute(0, 2, 1, 3, 4).reshape(S, N, s["q_heads"], D).to(out.dtype)
    return out[:-1]


# ------------------------------------------------------------------------------------------------ work
def work(case):
    D, Hk, b = case["dim"], case["kv_heads"], SIZE[case["type"]]
    if case["op"] == "norm_rope":
        n = case["tokens"] * (case["q_heads"] + Hk) * D
        return {"bytes": 2 * b * n + case["tokens"] * (4 * case["rot"] + 4) + 8 * D, "flops": 8 * n}
    new, ctx = _lengths(case, 1)
    fresh = sum(new)
    if case["op"] in ("write", "read"):
        return {"bytes": 2 * fresh * Hk * D * (b + 1) + 16 * sum(n // case["block"] + 1 for n in new) * Hk, "flops": 4 * fresh * Hk * D}
    w = case["window"] or 1 << 60
    keys = sum(min(c + n, n + w - 1) for n, c in zip(new, ctx))
    pairs = 0
    for n, c in zip(new, ctx):                                  # sum over i < n of min(c + i + 1, w)
        full = max(0, min(n, w - c))                            # queries that see everything before them
        pairs += full * c + full * (full + 1) // 2 + (n - full) * min(w, c + n)
    return {"bytes": 2 * keys * Hk * (D + 4 / case["block"]) + 2 * fresh * case["q_heads"] * D * b,
            "flops": 4 * pairs * case["q_heads"] * D}


# ------------------------------------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"norm_rope": _exact_norm_rope, "write": _exact_write, "read": _exact_read, "attn": _exact_attn}[case["op"]](s)


def _exact_norm_rope(s):
    ang = s["cs"][s["pos"].long()].double()
    turn = torch.complex(ang[..., 0], ang[..., 1])[:, None]
    res = {}
    for name, x, w in (("q", s["q"], s["q_w"]), ("k", s["k"], s["k_w"])):
        x = x.double()
        y = x / (x.pow(2).sum(-1, keepdim=True) / s["dim"] + EPS).sqrt() * w.double()
        i = torch.arange(s["rot"] // 2, device=x.device)
        at_a, at_b = (i, i + s["rot"] // 2) if s["halves"] else (2 * i, 2 * i + 1)
        z = torch.complex(y[..., s["first"] + at_a], y[..., s["first"] + at_b]) * turn
        y[..., s["first"] + at_a], y[..., s["first"] + at_b] = z.real, z.imag
        res[name] = y
    return res


def _e4m3(x):
    """x rounded to the nearest value of the format, ties to even mantissas."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _sequences(s):
    start, length = s["seq_start"].tolist(), s["kv_len"].tolist()
    for i in range(s["seqs"]):
        yield i, start[i], start[i + 1] - start[i], length[i]


def _exact_write(s):
    BT, res = s["block"], {}
    for name in "kv":
        val, sc = s[name + "_codes"].view(FP8).double(), s[name + "_scale"].double()
        for i, r, n, length in _sequences(s):
            p0 = length - n
            for b in range(p0 // BT, (length - 1) // BT + 1):
                lo, hi = max(p0, b * BT), min(length, b * BT + BT)
                blk = int(s["table"][i, b])
                x = s[name][r + lo - p0:r + hi - p0].double().transpose(0, 1)                     # [heads][rows][dim]
                amax = x.abs().amax((1, 2))
                e = torch.ceil(torch.log2((amax / 448).clamp(min=2.0 ** MIN_EXP)))
                e = torch.where(amax > 448 * torch.exp2(e), e + 1, torch.where(amax <= 448 * torch.exp2(e - 1), e - 1, e)).clamp(MIN_EXP, MAX_EXP)
                at = lo - b * BT
                if at:
                    e = torch.maximum(e, torch.log2(sc[blk]).round())
                    val[blk, :, :at] = _e4m3(val[blk, :, :at] * (sc[blk] / torch.exp2(e))[:, None, None])
                val[blk, :, at:at + hi - lo] = _e4m3((x / torch.exp2(e)[:, None, None]).clamp(-448, 448))
                sc[blk] = torch.exp2(e)
        res[name], res[name + "_scale"] = val, sc
    return res


def _exact_rows(s, name, i, lo, hi):
    """Values of positions [lo, hi) of sequence i: [heads][hi - lo][dim]."""
    b0, b1 = lo // s["block"], -(-hi // s["block"])
    ids = s["table"][i, b0:b1].long()
    x = s[name + "_codes"][ids].view(FP8).double() * s[name + "_scale"][ids].double()[:, :, None, None]
    return x.transpose(0, 1).flatten(1, 2)[:, lo - b0 * s["block"]:hi - b0 * s["block"]]


def _exact_read(s):
    res = {}
    for name in "kv":
        y = s[name + "_out"].double()
        for i, r, n, length in _sequences(s):
            y[r:r + n] = _exact_rows(s, name, i, length - n, length).transpose(0, 1)
        res[name] = y
    return res


def _exact_attn(s):
    out, G = s["out"].double(), s["q_heads"] // s["kv_heads"]
    for i, r, n, length in _sequences(s):
        k, v = _exact_rows(s, "k", i, 0, length), _exact_rows(s, "v", i, 0, length)
        pos = torch.arange(length - n, length, device=out.device)[:, None]
        at = torch.arange(length, device=out.device)
        hidden = (at > pos) | ((at <= pos - s["window"]) if s["window"] else False)
        for h in range(s["q_heads"]):
            logit = (s["q"][r:r + n, h].double() @ k[h // G].T / s["dim"] ** 0.5).masked_fill(hidden, -torch.inf)
            if s["sink"] is not None:
                logit = torch.cat([logit, s["sink"][h].double().expand(n, 1)], 1)
            out[r:r + n, h] = torch.softmax(logit, 1)[:, :length] @ v[h // G]
    return out
