"""Statements in 64 bits, on the CPU, of the operators whose rows choose their weights."""
import math

import torch

TYPES = {"float": torch.float32, "bfloat16": torch.bfloat16, "half": torch.float16}


def route(logits, bias, k, score, groups=1, top_groups=1, group_best=1, renormalise=False, scale=1.0):
    """(experts, weights in 64 bits), token by token"""
    ids, weights = [], []
    for x in logits.double():
        e = len(x)
        if score == "softmax":
            top = float(x[~x.isnan()].max()) if bool((~x.isnan()).any()) else -math.inf
            if top == -math.inf and not bool(x.isnan().any()):
                s = torch.zeros_like(x)
            else:
                z = (x - top).exp()
                s = z / z.sum()
        else:
            s = 1.0 / (1.0 + (-x).exp())
        rank = s if bias is None else s + bias.double()
        rank = torch.where(rank.isnan(), -math.inf, rank).tolist()
        allowed = set(range(e))
        if groups > 1:
            size = e // groups
            value = []
            for g in range(groups):
                best = sorted(rank[g * size:(g + 1) * size], reverse=True)[:group_best]
                v = sum(best)
                value.append(-math.inf if math.isnan(v) else v)
            kept = sorted(range(groups), key=lambda g: (-value[g], g))[:top_groups]
            allowed = {g * size + i for g in kept for i in range(size)}
        order = sorted(allowed, key=lambda i: (-rank[i], i))[:k]
        w = s[order]
        if renormalise:
            total = w.sum()
            w = torch.zeros_like(w) if float(total) == 0.0 else w / total
        ids.append(order)
        weights.append(w * scale)
    return torch.tensor(ids, dtype=torch.int32), torch.stack(weights)


def order(group_of, groups):
    """(offsets, rows)"""
    key = [g if 0 <= g < groups else groups for g in group_of.reshape(-1).tolist()]
    rows = sorted(range(len(key)), key=lambda i: (key[i], i))
    offsets = [sum(1 for v in key if v < g) for g in range(groups + 1)]
    return torch.tensor(offsets, dtype=torch.int32), torch.tensor(rows, dtype=torch.int32)


def quantize(x):
    """(codes, scale of each row) in 64 bits; scale NaN for a row that holds an infinity or NaN"""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    s = torch.maximum((top / 127.0).float(), torch.tensor(2.0 ** -100)).double()
    bad = ~torch.isfinite(x).all(-1, keepdim=True)
    codes = torch.where(bad, torch.zeros_like(x), (x / s).round())
    return codes, torch.where(bad, torch.full_like(s, math.nan), s)


def activate(name, x):
    if name == "swish":
        return x * torch.sigmoid(x)
    if name == "gelu_approx":
        return 0.5 * x * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (x + 0.044715 * x ** 3)))
    if name == "gelu_exact":
        return 0.5 * x * (1.0 + torch.erf(x / math.sqrt(2.0)))
    return x.clamp(min=0.0) if name == "relu" else x


def up(x, offsets, rows, top_k, w, scales, activation, gated):
    """w: codes [experts, each, N, K].  (h in 64 bits by place, NaN behind the last group; |gate|, |up| to weigh errors by)"""
    codes, s = quantize(x)
    h = torch.full((len(rows), w.shape[2]), math.nan, dtype=torch.float64)
    at = offsets.tolist()
    for e in range(w.shape[0]):
        if at[e] == at[e + 1]:
            continue
        token = rows[at[e]:at[e + 1]].long() // top_k
        v = [codes[token] @ w[e, i].double().T * s[token] * scales[e, i].double() for i in range(w.shape[1])]
        y = activate(activation, v[0])
        h[at[e]:at[e + 1]] = y * v[1] if gated else y
    return h


def down(h, experts, offsets, rows, w, scales, weights, addend):
    """(out in 64 bits, the sum of its parts' absolute values)"""
    tokens, k = experts.shape
    codes, s = quantize(h)
    n = w.shape[2]
    y = torch.zeros(tokens * k, n, dtype=torch.float64)
    at = offsets.tolist()
    for e in range(w.shape[0]):
        places = torch.arange(at[e], at[e + 1])
        y[rows[places].long()] = codes[places] @ w[e, 0].double().T * s[places] * scales[e, 0].double()
    y = y.reshape(tokens, k, n)
    there = ((experts >= 0) & (experts < w.shape[0]))[..., None]
    parts = torch.where(there, y * weights.double()[..., None], torch.zeros((), dtype=torch.float64))
    out = parts.sum(1)
    size = parts.abs().sum(1)
    if addend is not None:
        out, size = out + addend.double(), size + addend.double().abs()
    return out, size


def adapters(x, offsets, rows, a, b, ranks, scales, base, slice_ends, rank):
    """(out in 64 bits, what its terms add up to in absolute value: |base|, and scale |x| |A|^T |B|^T)"""
    out, size = base.double().clone(), base.double().abs()
    at = offsets.tolist()
    for g in range(a.shape[0]):
        t = rows[at[g]:at[g + 1]].long()
        if len(t) == 0:
            continue
        r = rank if ranks is None else min(max(int(ranks[g]), 0), rank)
        begin = 0
        for i, end in enumerate(slice_ends):
            left, right = a[g].double()[i * rank:i * rank + r], b[g].double()[begin:end, :r]
            out[t, begin:end] += float(scales[g]) * ((x[t].double() @ left.T) @ right.T)
            size[t, begin:end] += abs(float(scales[g])) * ((x[t].double().abs() @ left.abs().T) @ right.abs().T)
            begin = end
    return out, size
