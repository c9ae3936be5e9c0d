"""Plain 64-bit statements of the operators between a decoder's qkv linear and its output linear, for the tests: written from the
formulas in include/itexhip.h, on the CPU, a row at a time."""
import math

import torch


def padded(d):
    return 64 if d <= 64 else 128 if d <= 128 else 256


def norm_rope(x, weight, eps, positions, freqs, rotary_dim, interleaved, factor):
    """x [tokens, heads, d]; freqs in turns a position"""
    y = x.double().clone()
    if weight is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * weight.double()
    if rotary_dim == 0:
        return y
    turns = positions.double()[:, None] * freqs.double()[None, :]
    angle = (turns - turns.round()) * (2.0 * math.pi)
    c, s = angle.cos()[:, None, :] * factor, angle.sin()[:, None, :] * factor
    i = torch.arange(rotary_dim // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rotary_dim // 2)
    out = y.clone()
    out[..., a] = y[..., a] * c - y[..., b] * s
    out[..., b] = y[..., b] * c + y[..., a] * s
    return out


def quantize(x):
    """codes 0 .. 15, scale and offset (float64 holding halves) of [..., d]"""
    x = x.clamp(-65504.0, 65504.0)
    hi, lo = x.amax(-1, keepdim=True), x.amin(-1, keepdim=True)
    scale = ((hi - lo) / 15.0).float().half().double()
    offset = (lo + 8.0 * scale).float().half().double()
    code = torch.where(scale == 0, torch.zeros_like(x), torch.round((x - offset) / torch.where(scale == 0, torch.ones_like(scale), scale)))
    bad = torch.isnan(x).any(-1, keepdim=True)
    scale, offset = torch.where(bad, math.nan, scale), torch.where(bad, math.nan, offset)
    return torch.where(bad, torch.zeros_like(code), code).clamp(-8, 7).to(torch.int64) + 8, scale, offset


def values(code, scale, offset):
    return scale * (code - 8).double() + offset


class Cache:
    """Pages as include/itexhip.h lays them out, with random codes and parameters at the slots in `used`; the others hold whatever
    memory held: any codes, parameters NaN, infinite or huge."""

    def __init__(self, pages, heads, d, page_size, used, seed=0, scale=0.36, offset=0.3):
        g = torch.Generator().manual_seed(seed)
        n = pages * page_size
        self.pages, self.heads, self.d, self.p, self.dp = pages, heads, d, page_size, padded(d)
        self.code = torch.randint(0, 16, (2, n, heads, d), generator=g)
        self.scale = (torch.exp(0.3 * torch.randn(2, n, heads, generator=g)) * scale).half().double()
        self.offset = (torch.randn(2, n, heads, generator=g) * offset).half().double()
        stale = torch.ones(n, dtype=torch.bool)
        stale[torch.as_tensor(list(used), dtype=torch.int64)] = False
        junk = torch.tensor([math.nan, math.inf, -math.inf, 65504.0], dtype=torch.float64)
        self.scale[:, stale] = junk[torch.randint(0, 4, (2, int(stale.sum()), heads), generator=g)]
        self.offset[:, stale] = junk[torch.randint(0, 4, (2, int(stale.sum()), heads), generator=g)]

    @property
    def k(self):
        return values(self.code[0], self.scale[0][..., None], self.offset[0][..., None])

    @property
    def v(self):
        return values(self.code[1], self.scale[1][..., None], self.offset[1][..., None])

    def pack(self):
        n, h, p, pages, dp = self.pages * self.p, self.heads, self.p, self.pages, self.dp
        full = torch.full((2, n, h, dp), 8, dtype=torch.int64)
        full[..., :self.d] = self.code
        byte = (full[..., 0::2] | (full[..., 1::2] << 4)).to(torch.uint8)
        keys = byte[0].reshape(pages, p, h, dp // 2).permute(0, 2, 1, 3).reshape(pages, h, -1)
        vals = byte[1].reshape(pages, p // 4, 4, h, dp // 8, 4).permute(0, 3, 1, 4, 2, 5).reshape(pages, h, -1)
        par = torch.stack([self.scale, self.offset], -1).to(torch.float16).reshape(2, pages, p // 4, 4, h, 2).permute(0, 1, 4, 2, 5, 3)
        par = par.contiguous().view(torch.uint8).reshape(2, pages, h, -1)
        return torch.cat([keys, vals, par[0], par[1]], -1).contiguous()


def attention(q, cache, table, cu_q, kv_len, scale, causal=True, window=0):
    """(out, lse, mass): mass bounds sum p |scale code| + p |offset| over a row's dimensions, what roundings of p are relative to.
    q [rows, heads, d]"""
    rows, hq, d = q.shape
    group = hq // cache.heads
    out, lse, mass = torch.zeros(rows, hq, d, dtype=torch.float64), torch.full((rows, hq), -math.inf, dtype=torch.float64), torch.zeros(rows, hq, dtype=torch.float64)
    pages, keys, vals = cache.pages, cache.k, cache.v
    for b, n in enumerate(kv_len):
        m = cu_q[b + 1] - cu_q[b]
        n = min(n, len(table[b]) * cache.p)
        for i in range(m):
            pos = n - m + i
            seen = [t for t in range(n) if (not causal or t <= pos) and (not window or t > pos - window) and 0 <= table[b][t // cache.p] < pages]
            if not seen:
                continue
            slots = torch.tensor([table[b][t // cache.p] * cache.p + t % cache.p for t in seen])
            for h in range(hq):
                k, v = keys[slots, h // group], vals[slots, h // group]
                z = (k * q[cu_q[b] + i, h].double()).sum(-1) * scale
                top = z.max()
                p = (z - top).exp()
                l = p.sum()
                out[cu_q[b] + i, h] = (p[:, None] * v).sum(0) / l
                lse[cu_q[b] + i, h] = top + l.log()
                mass[cu_q[b] + i, h] = (p * (8.0 * cache.scale[1][slots, h // group] + cache.offset[1][slots, h // group].abs())).sum() / l
    return out, lse, mass
