"""The 8-bit cache, head norms with rotation and attention over the cache in 64 bits, as their definitions say, and batches for tests."""
import numpy as np
import torch

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
FP8 = torch.float8_e4m3fn


def half_step(dt):
    """A rounding's relative error, and what a value below the normal range may be off by."""
    return torch.finfo(dt).eps / 2, torch.finfo(dt).smallest_normal * torch.finfo(dt).eps / 2


def e4m3(x):
    """float64 -> nearest e4m3 value, ties to even, beyond the format: the largest."""
    x = x.clamp(-448, 448)                                           # first: the step of an infinity is none
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def values(codes):
    return codes.view(FP8).to(torch.float64)


class Case:
    """Sequences of (new, len) over a cache whose other blocks, rows and table entries hold garbage."""

    def __init__(self, seqs, kv_heads, dim, block, seed, pad=0, device="cuda", spare=2):
        g = torch.Generator().manual_seed(seed)
        self.seqs, self.kv_heads, self.dim, self.block, self.device, self.g = seqs, kv_heads, dim, block, device, g
        per = max(1, max(-(-l // block) for _, l in seqs)) + 1
        n = len(seqs) * per + spare
        order = torch.randperm(n, generator=g)
        junk = torch.tensor([-1, n, 2 ** 31 - 1, -2 ** 31, n + 7], dtype=torch.int64)
        table = junk[torch.randint(0, 5, (len(seqs), per), generator=g)]
        used = torch.zeros(n, dtype=torch.bool)
        k = 0
        for s, (_, l) in enumerate(seqs):
            for b in range(-(-l // block)):
                table[s, b] = order[k]
                used[order[k]] = True
                k += 1
        start = np.cumsum([0] + [a for a, _ in seqs])
        self.rows = int(start[-1]) + pad
        shape = (n, kv_heads, block, dim)

        def codes():
            x = (torch.randn(shape, generator=g) * 112).clamp(-448, 448).to(FP8).view(torch.uint8)
            x[~used] = 0x7F                                            # NaN
            for s, (_, l) in enumerate(seqs):
                if l % block:
                    x[table[s, l // block], :, l % block:] = 0xFF
            return x.to(device)

        def scales():
            x = torch.exp2(torch.randint(-9, -5, shape[:2], generator=g).float())
            x[~used] = float("nan")
            return x.to(device)
        self.k, self.v, self.ks, self.vs = codes(), codes(), scales(), scales()
        self.table_host = table
        self.table = table.to(torch.int32).to(device)
        self.start, self.start_host = torch.tensor(start, dtype=torch.int32, device=device), [int(v) for v in start]
        self.len = torch.tensor([l for _, l in seqs], dtype=torch.int32, device=device)
        self.max_new, self.max_len = max(1, max(a for a, _ in seqs)), max(1, max(l for _, l in seqs))
        self.rows = max(self.rows, self.max_new)

    def cache(self):
        from macseek_b200 import kv8
        return kv8.Cache.of(self.k, self.v, self.ks, self.vs)

    def batch(self, **kw):
        from macseek_b200 import kv8
        a = dict(n_tokens=self.rows, max_new=self.max_new, max_len=self.max_len)
        a.update(kw)
        return kv8.Batch(self.start, self.len, self.table, **a)

    def randn(self, *shape, dt="f32", mul=1.0):
        return (torch.randn(shape, generator=self.g) * mul).to(DT[dt]).to(self.device)

    def held(self, s, which, lo=0):
        """float64 [kv_heads][len - lo][dim] of sequence s."""
        codes, scale = (self.k, self.ks) if which == "k" else (self.v, self.vs)
        l = self.seqs[s][1]
        ids = self.table_host[s, :-(-l // self.block)].to(codes.device)
        x = values(codes[ids]) * scale[ids].double()[:, :, None, None]
        return x.transpose(0, 1).flatten(1, 2)[:, lo:l]


def write_ref(c, k, v):
    """(codes' values, scale) of keys and of values after the rows are written; untouched bytes stay as they are."""
    res = []
    for x, codes, scale in ((k, c.k, c.ks), (v, c.v, c.vs)):
        val, sc = values(codes), scale.double().clone()
        for s, (n, l) in enumerate(c.seqs):
            p0 = l - n
            for b in range(p0 // c.block, -(-l // c.block) if n else 0):
                lo, hi = max(p0, b * c.block), min(l, (b + 1) * c.block)
                blk = int(c.table_host[s, b])
                rows = x[c.start_host[s] + lo - p0:c.start_host[s] + hi - p0].double().transpose(0, 1)
                rows = torch.where(torch.isnan(rows), torch.zeros_like(rows), rows)
                top = torch.where(torch.isinf(rows), torch.zeros_like(rows), rows).abs().amax((1, 2))
                e = torch.full_like(top, -50)
                for t in range(-50, 50):                                        # the smallest that holds it
                    e = torch.where(top > 448 * 2.0 ** t, torch.full_like(e, t + 1), e)
                at = lo - b * c.block
                if at:
                    old = torch.log2(sc[blk]).round()
                    e = torch.maximum(e, old)
                    val[blk, :, :at] = e4m3(val[blk, :, :at] * torch.exp2(old - e)[:, None, None])
                val[blk, :, at:at + hi - lo] = e4m3(rows * torch.exp2(-e)[:, None, None])
                sc[blk] = torch.exp2(e)
        res += [val, sc]
    return res


def attn_ref(c, q, out0, scale, window=0, sinks=None):
    """(out, tolerance per element) in float64.  The tolerance, for a row that sees L tokens, A = scale * max_j sum |q_i k_ji| and
    V = max |v|: a logit is off by d = A ((D / 8 + 16) 2^-22 + 2^-21) (products added 16 at a time in 32 bits, the query as halves);
    weights by 2.2 d + 2^-20 (2^x within two units) and their own rounding (2^-11, F32: 2^-21, and 2^-25 of the largest one); sums over L
    tokens by (L / 8 + 32) 2^-23; all times V, and the output is rounded once."""
    out, tol = out0.double().clone(), torch.zeros_like(out0, dtype=torch.float64)
    heads, D = q.shape[1], q.shape[2]
    G = heads // c.kv_heads
    half, tiny = half_step(q.dtype)
    two = q.dtype == torch.float32
    for s, (n, l) in enumerate(c.seqs):
        if n == 0:
            continue
        k, v = c.held(s, "k"), c.held(s, "v")
        r = slice(c.start_host[s], c.start_host[s] + n)
        pos = torch.arange(l - n, l, device=q.device)[:, None]
        at = torch.arange(l, device=q.device)
        seen = at <= pos
        if window:
            seen &= at > pos - window
        L = seen.sum(1, keepdim=True).double()
        for h in range(heads):
            x = q[r, h].double()
            lg = (x @ k[h // G].T) * scale
            A = torch.where(seen, (x.abs() @ k[h // G].abs().T) * abs(scale), 0.0).amax(1, keepdim=True)
            lg = lg.masked_fill(~seen, -torch.inf)
            if sinks is not None:
                lg = torch.cat([lg, sinks[h].double().expand(n, 1)], 1)
            ref = torch.softmax(lg, 1)[:, :l] @ v[h // G]
            V = torch.where(seen[:, :, None], v[h // G].abs()[None], 0.0).amax(1) if n * l * D < 3e7 else v[h // G].abs().amax(0)[None]
            d = A * ((D / 8 + 16) * 2.0 ** -22 + 2.0 ** -21)
            e = 2.2 * d + 2.0 ** -20 + (2.0 ** -21 if two else 2.0 ** -11 + L * 2.0 ** -25) + (L / 8 + 32) * 2.0 ** -23
            out[r, h] = ref
            tol[r, h] = V * e * (1 + half) + half * ref.abs() + tiny
    return out, tol


def norm_rope_ref(x, w, eps, cs, pos, first, halves):
    """(out, tolerance) in float64: the norm is off by less than 20 units of 2^-24 (a sum of D squares by eights and halves, a root,
    two products), a rotated value by 4 more of each product, and the output is rounded once."""
    x = x.double()
    y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * (1.0 if w is None else w.double())
    mag, out = y.abs().clone(), y.clone()
    half = cs.shape[1]
    i = torch.arange(half, device=x.device)
    ia, ib = (first + i, first + i + half) if halves else (first + 2 * i, first + 2 * i + 1)
    f = cs[pos.clamp(min=0).long()].double()[:, None]
    a, b = y[..., ia], y[..., ib]
    out[..., ia], out[..., ib] = a * f[..., 0] - b * f[..., 1], a * f[..., 1] + b * f[..., 0]
    mag[..., ia], mag[..., ib] = (a * f[..., 0]).abs() + (b * f[..., 1]).abs(), (a * f[..., 1]).abs() + (b * f[..., 0]).abs()
    return out, mag * 24 * 2.0 ** -24
