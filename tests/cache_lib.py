"""What the tests of the paged cache and its attention share: the definitions in float64, and a cache with sequences in it."""
import math

import numpy as np
import torch

TDT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
LIMIT = {"f16": 65504.0, "bf16": 3.3895313892515355e38, "q8": 57344.0, "q4": 57344.0}


def held(kind, x):
    """What a cache of this kind holds for fp32 x [..., dim], as float64."""
    x = torch.nan_to_num(x.float(), nan=0.0, posinf=math.inf, neginf=-math.inf).clamp(-LIMIT[kind], LIMIT[kind])
    if kind in TDT:
        return x.to(TDT[kind]).double()
    top = 127.0 if kind == "q8" else 7.0
    g = x.unflatten(-1, (-1, 32))
    d = (g.abs().amax(dim=-1).double() / top).float().half()                 # (a quotient of two fp32 numbers rounded twice is rounded once)
    r = (g.double() / d.double().unsqueeze(-1)).float().double()
    q = torch.where(d.unsqueeze(-1) == 0, 0.0, torch.sign(r) * torch.floor(r.abs() + 0.5)).clamp(-top, top)
    return (q * d.double().unsqueeze(-1)).flatten(-2)


def rope_table(positions, dims, base=10000.0):
    angle = np.arange(positions)[:, None] * base ** (-np.arange(0, dims, 2) / dims)
    return torch.from_numpy(np.stack([np.cos(angle), np.sin(angle)], axis=2).astype(np.float32)).cuda()


def turned(x, positions, rope, style):
    """fp64 sums of exact products, rounded to fp32; rows without a position (below 0, behind the table) come back unturned."""
    if rope is None:
        return x.float()
    dims = rope.shape[1] * 2
    p = torch.as_tensor(positions, device="cuda").clamp(0, rope.shape[0] - 1)
    c, s = (rope[p][:, :, i].double().unsqueeze(1) for i in range(2))
    x = x.double()
    out = x.clone()
    a, b = (slice(0, dims // 2), slice(dims // 2, dims)) if style == "halves" else (slice(0, dims, 2), slice(1, dims, 2))
    out[:, :, a] = x[:, :, a] * c - x[:, :, b] * s
    out[:, :, b] = x[:, :, b] * c + x[:, :, a] * s
    return out.float()


def normal(shape, seed, dt="f32", std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.empty(shape, device="cuda").normal_(0.0, std, generator=g).to(TDT[dt])


class Cached:
    """Sequences of `lengths` tokens in a cache, in pages in no order; `k`, `v` [tokens, kv heads, dim]: what they hold, in float64."""

    def __init__(self, be, kind, lengths, kv_heads=2, dim=128, page=64, seed=1, dt=None, layers=1, layer=0, width=None, spare=1):
        self.be, self.kind, self.lengths, self.kv_heads, self.dim, self.page, self.layer = be, kind, list(lengths), kv_heads, dim, page, layer
        dt = dt or (kind if kind in TDT else "f16")
        per = [-(-n // page) for n in lengths]
        self.cache = be.kv_cache(kind, layers, kv_heads, dim, page, max(1, sum(per) + spare))
        order = np.random.default_rng(seed).permutation(self.cache.pages)
        self.tables = torch.full((len(lengths), max(1, width or max(per))), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(per):
            self.tables[b, :n] = torch.from_numpy(order[at:at + n].astype(np.int32))
            at += n
        self.tables = self.tables.cuda()
        total = sum(lengths)
        self.k_in, self.v_in = normal((total, kv_heads, dim), seed + 1, dt), normal((total, kv_heads, dim), seed + 2, dt)
        self.k, self.v = held(kind, self.k_in), held(kind, self.v_in)
        if total:
            be.cache_append(self.cache, layer, self.batch(self.lengths), None, self.k_in, self.v_in)
        torch.cuda.synchronize()

    def batch(self, new, rows=None, lengths=None, max_new=None):
        ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
        starts = np.concatenate([[0], np.cumsum(new)]).tolist()
        return self.be.cache_batch(ints(starts), ints(self.lengths if lengths is None else lengths), self.tables,
                                   rows if rows is not None else int(sum(new)), max_new or max(1, max(new)))

    def expected(self, q, new, scale=None, window=0, hidden=lambda b, j: False):
        """float64 y of rows q [rows, heads, dim], and the sums of p |v| and the largest |q| |k| scale that its error hangs on."""
        heads = q.shape[1]
        group, scale = heads // self.kv_heads, self.dim ** -0.5 if scale is None else scale
        y = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
        size, dots = torch.zeros_like(y), torch.zeros(q.shape[:2] + (1,), dtype=torch.float64, device="cuda")
        row = token = 0
        for n, L, b in zip(new, self.lengths, range(len(new))):
            if n and L:
                p = torch.arange(L - n, L, device="cuda").reshape(-1, 1)
                j = torch.arange(L, device="cuda")
                gone = torch.tensor([hidden(b, int(x)) for x in range(L)], device="cuda")
                seen = (j <= p) & ~gone
                if window:
                    seen &= j > p - window
                for h in range(heads):
                    k, v = (t[token:token + L, h // group] for t in (self.k, self.v))
                    qq = q[row:row + n, h].double()
                    s = torch.where(seen, qq @ k.T.contiguous() * scale, -math.inf)
                    top = s.amax(dim=1, keepdim=True)
                    e = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
                    e = e / e.sum(dim=1, keepdim=True).clamp(min=1e-300)
                    y[row:row + n, h] = e @ v
                    size[row:row + n, h] = e @ v.abs()
                    dots[row:row + n, h, 0] = torch.where(seen, qq.abs() @ k.abs().T.contiguous() * scale, 0.0).amax(dim=1)
            row += n
            token += L
        return y, size, dots

    def close(self):
        self.cache.free()
