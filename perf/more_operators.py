"""Linears whose weights a token chooses, as cases that can be timed and compared: routing to experts, the experts' quantized
products, low-rank adapters beside a shared projection.

kind        one pass
route       scores of a router's logits, the experts and weights of each token, and the order of their rows by expert
up          rows of activations quantized each by its own largest value, the products of each row's expert, the activation between
            gate and up
down        rows of the experts' hidden values quantized the same way, the products, and each token's weighted sum of its experts
adapters    out = base + scale * (x A^T) B^T with the A and B of each token's adapter, columns in one or several slices

The order of rows: `offsets` [groups + 1] and `rows`, a permutation of the slots (token * top_k + choice) that lists them by group,
within a group by slot, and those that chose no group of this device at the end.

A row's codes: scale = max(largest absolute value / 127, 2^-100) as a 32-bit float, code = the quotient by it, rounded half to even.
"""
import importlib
import math
import random

import torch

own = False

_TORCH = {"float": torch.float32, "bfloat16": torch.bfloat16, "half": torch.float16}
_BYTES = {"float": 4, "bfloat16": 2, "half": 2}


def listed():
    return [
        # one new token of a decoder with 8 experts: latency
        dict(name="route_1", kind="route", T=1, E=8, k=2, score="softmax", groups=1, top_groups=1, best=1, bias=False, renorm=True, scale=1.0, type="bfloat16"),
        # 64 served sequences, many small experts
        dict(name="route_64", kind="route", T=64, E=64, k=6, score="softmax", groups=1, top_groups=1, best=1, bias=False, renorm=False, scale=1.0, type="half"),
        # a prompt, experts in groups that are chosen first, a bias that balances their load
        dict(name="route_8192", kind="route", T=8192, E=256, k=8, score="sigmoid", groups=8, top_groups=4, best=2, bias=True, renorm=True, scale=2.5, type="float"),
        # the next token through its two experts of an 8B decoder's linears: both weights are read once
        dict(name="up_1", kind="up", T=1, E=8, k=2, K=4096, N=14336, gated=True, act="swish", part=False, type="bfloat16"),
        # 64 served sequences, small experts, of which nearly all are read
        dict(name="up_64", kind="up", T=64, E=64, k=6, K=2048, N=1408, gated=True, act="swish", part=False, type="half"),
        # a prompt
        dict(name="up_4096", kind="up", T=4096, E=8, k=2, K=4096, N=14336, gated=True, act="swish", part=False, type="bfloat16"),
        # the way back of the next token
        dict(name="down_1", kind="down", T=1, E=8, k=2, K=14336, N=4096, addend=True, part=False, type="bfloat16"),
        # a ragged number of tokens, half of the experts on another device, odd sizes, fp32
        dict(name="down_333_odd", kind="down", T=333, E=12, k=4, K=1000, N=770, addend=False, part=True, type="float"),
        # a prompt's way back
        dict(name="down_4096", kind="down", T=4096, E=8, k=2, K=14336, N=4096, addend=True, part=False, type="bfloat16"),
        # one request with an adapter of its own: latency
        dict(name="adapters_1", kind="adapters", T=1, A=8, R=16, K=4096, slices="4096", ragged=False, type="bfloat16"),
        # 64 requests, hardly two with the same adapter, queries, keys and values in one projection
        dict(name="adapters_64", kind="adapters", T=64, A=64, R=16, K=4096, slices="4096 1024 1024", ragged=True, type="half"),
        # prompts of several requests, wide linear
        dict(name="adapters_8192", kind="adapters", T=8192, A=5, R=64, K=4096, slices="14336", ragged=False, type="bfloat16"),
    ]


def _log(rng, lo, hi):
    """A size between lo and hi, even over its logarithm."""
    return max(1, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi)))))))


def draw(rng):
    kind = rng.choice(["route", "up", "down", "adapters", "adapters"])
    t = rng.choice(["bfloat16", "half", "float"])
    if kind == "route":
        e = rng.choice([4, 8, 16, 60, 64, 96, 128, 160, 256])
        groups = rng.choice([g for g in (1, 1, 4, 8) if e % g == 0])
        top_groups = 1 if groups == 1 else rng.randint(1, groups)
        return dict(kind="route", T=_log(rng, 1, 8192), E=e, k=rng.randint(1, min(8, top_groups * e // groups)), score=rng.choice(["softmax", "sigmoid"]),
                    groups=groups, top_groups=top_groups, best=rng.choice([1, 2]) if groups > 1 and e // groups > 1 else 1, bias=rng.choice([True, False]),
                    renorm=rng.choice([True, False]), scale=rng.choice([1.0, 1.0, 2.5]), type=t)
    if kind == "adapters":
        slices = rng.choice([str(16 * _log(rng, 8, 896)), "4096 1024 1024", "768 768 768", "2048 256 256", "1408 1408"])
        tokens = _log(rng, 1, 8192 if t != "float" else 2048)
        return dict(kind="adapters", T=tokens, A=_log(rng, 1, 64), R=rng.choice([8, 16, 16, 32, 64]), K=8 * _log(rng, 16, 512),
                    slices=slices, ragged=rng.choice([True, False]), type=t)
    e = rng.choice([4, 8, 8, 16, 32, 64, 128])
    k = rng.randint(1, min(8, e))
    tokens = _log(rng, 1, 4096)
    most = min(8 * 4096 * 14336 // e, 4096 * 2 * 4096 * 14336 // (tokens * k))      # elements of one expert's weight
    a = rng.choice([512, 768, 1000, 1408, 2048, 4096])
    b = max(16, min(14336, _log(rng, 256, max(256, most // a))))
    b = min(b if rng.random() < 0.3 else max(16, b // 16 * 16), max(16, most // a))
    if kind == "up":
        gated = rng.choice([True, True, False])
        return dict(kind="up", T=tokens, E=e, k=k, K=a, N=b, gated=gated, act=rng.choice(["swish", "swish", "gelu", "relu"]), part=rng.choice([True, False, False]), type=t)
    return dict(kind="down", T=tokens, E=e, k=k, K=b, N=a, addend=rng.choice([True, False]), part=rng.choice([True, False, False]), type=t)


# ---------------------------------------------------------------------------------------------------------------------
# what a program has in hand before the call
# ---------------------------------------------------------------------------------------------------------------------
def _order(chosen, groups):
    """(offsets, rows) of the slots that chose groups 0 .. groups - 1; the other slots come last."""
    key = torch.where((chosen < 0) | (chosen >= groups), groups, chosen).reshape(-1).long()
    rows = torch.sort(key, stable=True)[1].to(torch.int32)
    counts = (key[:, None] == torch.arange(groups, device=key.device)).sum(0)
    return torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32), rows


def _choices(case, g):
    """k different experts of each token, some more liked than others; with `part` as many again are on another device."""
    total = case["E"] * (2 if case["part"] else 1)
    liked = torch.randn(1, total, device="cuda", generator=g) * 0.5
    return (torch.randn(case["T"], total, device="cuda", generator=g) + liked).topk(case["k"], -1)[1].to(torch.int32)


def _slices(case):
    return [int(n) for n in case["slices"].split()]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = dict(case)
    t, n = _TORCH[case["type"]], case["T"]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    if case["kind"] == "route":
        s["logits"] = (normal(n, case["E"]) * 1.5 + normal(1, case["E"]) * 0.5).to(t)
        s["bias_of"] = normal(case["E"]) * 0.1 if case["bias"] else None
        s["experts"] = torch.empty(n, case["k"], dtype=torch.int32, device="cuda")
        s["weights"] = torch.empty(n, case["k"], device="cuda")
        s["offsets"] = torch.empty(case["E"] + 1, dtype=torch.int32, device="cuda")
        s["rows"] = torch.empty(n * case["k"], dtype=torch.int32, device="cuda")
    elif case["kind"] == "adapters":
        a, r, out = case["A"], case["R"], sum(_slices(case))
        spread = (normal(1, case["K"]) * 0.25).exp_()
        s["x"] = (normal(n, case["K"]) * spread).to(t)
        s["base"] = normal(n, out).to(t)                                             # the shared projection's output
        s["a"] = (normal(a, len(_slices(case)) * r, case["K"]) * case["K"] ** -0.5).to(t)
        s["b"] = (normal(a, out, r) * 0.05).to(t)
        s["scales"] = 0.5 + torch.rand(a, device="cuda", generator=g)
        s["ranks"] = (r - 8 * torch.randint(0, r // 8, (a,), device="cuda", generator=g)).to(torch.int32) if case["ragged"] else None
        # runs of tokens of one request; with more requests than adapters some share one; one request in ten has none
        requests = min(n, max(1, n if n <= 64 else 2 * a))
        of = torch.randint(0, a, (requests,), device="cuda", generator=g)
        of[torch.rand(requests, device="cuda", generator=g) < 0.1] = -1
        if n == 1:
            of[:] = a - 1
        request = torch.sort(torch.randint(0, requests, (n,), device="cuda", generator=g))[0] if n > requests else torch.arange(n, device="cuda")
        s["offsets"], s["rows"] = _order(of[request], a)
        s["starts"] = s["offsets"].tolist()
        s["out"] = torch.empty_like(s["base"])
    else:
        e, k, up = case["E"], case["k"], case["kind"] == "up"
        each = 2 if up and case["gated"] else 1
        s["experts"] = _choices(case, g)
        s["offsets"], s["rows"] = _order(s["experts"], e)
        s["starts"] = s["offsets"].tolist()
        if up:
            s["x"] = (normal(n, case["K"]) * (normal(1, case["K"]) * 0.25).exp_()).to(t)
            s["h"] = torch.zeros(n * k, case["N"], dtype=t, device="cuda")          # rows behind the last group stay
        else:
            v = normal(n * k, case["K"])
            s["h"] = (v * torch.sigmoid(v) * normal(n * k, case["K"])).to(t)
            s["weights"] = torch.softmax(normal(n, k), -1)
            s["residual"] = normal(n, case["N"]).to(t) if case["addend"] else None
            s["out"] = torch.empty(n, case["N"], dtype=t, device="cuda")
        s["w_scales"] = (0.8 + 0.4 * torch.rand(e, each, case["N"], device="cuda", generator=g)) * (0.03 / case["K"] ** 0.5)
        s["w"] = torch.empty(e, each, case["N"], case["K"], dtype=torch.int8, device="cuda")
        for i in range(e):
            s["w"][i] = (normal(each, case["N"], case["K"]) * 33.0).round_().clamp_(-127, 127).to(torch.int8)
    if own:
        _plan(s)
    return s


def _plan(s):
    """What a program that calls the framework keeps: its parameter structures, packed weights and workspaces."""
    hip = importlib.import_module("intel-extension-for-tensorflow_amd").itexhip
    t = {"float": hip.FLOAT, "bfloat16": hip.BFLOAT16, "half": hip.HALF}[s["type"]]
    s["hip"] = hip
    if s["kind"] == "route":
        s["params"] = hip.route_params(t, s["E"], s["k"], score=hip.ROUTE_SIGMOID if s["score"] == "sigmoid" else hip.ROUTE_SOFTMAX, groups=s["groups"],
                                       top_groups=s["top_groups"], group_best=s["best"], renormalise=s["renorm"], scale=s["scale"])
        size = hip.group_rows_workspace(s["T"] * s["k"], s["E"])
    elif s["kind"] == "adapters":
        ends = [sum(_slices(s)[:i + 1]) for i in range(len(_slices(s)))]
        s["params"] = hip.adapters_params(t, s["A"], s["R"], s["T"], s["K"], ends)
        size = hip.adapters_workspace(s["params"])
    else:
        up = s["kind"] == "up"
        act = {"swish": hip.ACT_SWISH, "gelu": hip.ACT_GELU_APPROX, "relu": hip.ACT_RELU}[s["act"]] if up else hip.ACT_NONE
        hidden, inner = (s["K"], s["N"]) if up else (s["N"], s["K"])
        s["params"] = hip.experts_params(t, s["E"], s["k"], s["T"], hidden, inner, activation=act, gated=up and s["gated"])
        size = hip.experts_workspace(s["params"])
        w = s.pop("w")
        e, each, n, k = w.shape
        s["packed"] = torch.empty(e, each, hip.qgemm_packed_bytes(k, n), dtype=torch.int8, device="cuda")
        sums = torch.empty(n, dtype=torch.int32, device="cuda")
        for i in range(e):
            for j in range(each):
                hip.qgemm_prepack_b(w[i, j], True, k, n, s["packed"][i, j], sums)
    s["workspace"] = torch.empty(size, dtype=torch.uint8, device="cuda")


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(s):
    if own:
        return _run_own(s)
    return {"route": _route, "up": _up, "down": _down, "adapters": _adapters}[s["kind"]](s)


def _run_own(s):
    hip = s["hip"]
    if s["kind"] == "route":
        hip.route(s["params"], s["T"], s["logits"], s["bias_of"], s["experts"], s["weights"])
        hip.group_rows(s["T"] * s["k"], s["E"], s["experts"], s["offsets"], s["rows"], s["workspace"])
        return {"experts": s["experts"], "weights": s["weights"], "offsets": s["offsets"], "rows": s["rows"]}
    if s["kind"] == "up":
        hip.experts_up(s["params"], s["x"], s["offsets"], s["rows"], s["packed"], s["w_scales"], s["h"], s["workspace"])
        return s["h"]
    if s["kind"] == "down":
        hip.experts_down(s["params"], s["h"], s["experts"], s["offsets"], s["rows"], s["packed"], s["w_scales"], s["weights"], s["residual"], s["out"], s["workspace"])
        return s["out"]
    hip.adapters(s["params"], s["x"], s["offsets"], s["rows"], s["a"], s["b"], s["ranks"], s["scales"], s["base"], s["out"], s["workspace"])
    return s["out"]


def _route(s):
    """Ranked in 64 bits: scores lie next to one another."""
    x = s["logits"].double()
    if s["score"] == "softmax":
        z = (x - x.amax(-1, keepdim=True)).exp()
        score = z / z.sum(-1, keepdim=True)
    else:
        score = 1.0 / (1.0 + (-x).exp())
    rank = score if s["bias_of"] is None else score + s["bias_of"].double()
    if s["groups"] > 1:
        of = rank.reshape(s["T"], s["groups"], -1)
        best = of.sort(dim=-1, descending=True)[0][..., :s["best"]].sum(-1)
        chosen = best.sort(dim=-1, descending=True, stable=True)[1][:, :s["top_groups"]]
        kept = (chosen[:, :, None] == torch.arange(s["groups"], device=x.device)).any(1)
        rank = torch.where(kept[..., None], of, -math.inf).reshape(s["T"], -1)
    experts = rank.sort(dim=-1, descending=True, stable=True)[1][:, :s["k"]]
    w = score.gather(-1, experts)
    if s["renorm"]:
        w = w / w.sum(-1, keepdim=True)
    offsets, rows = _order(experts, s["E"])
    return {"experts": experts.to(torch.int32), "weights": (w * s["scale"]).float(), "offsets": offsets, "rows": rows}


def _codes(x):
    """Codes (whole numbers, in 32 bits) and scale of each row; quotients in 64 bits, as they lie next to halves."""
    x = x.double()
    scale = (x.abs().amax(-1, keepdim=True) / torch.full((), 127.0, dtype=torch.float64, device=x.device)).float().clamp(min=2.0 ** -100)
    return (x / scale.double()).round().float(), scale


def _up(s):
    codes, scale = _codes(s["x"])
    h = torch.zeros(s["T"] * s["k"], s["N"], dtype=s["x"].dtype, device="cuda")
    for e in range(s["E"]):
        a, b = s["starts"][e], s["starts"][e + 1]
        if a == b:
            continue
        token = s["rows"][a:b].long() // s["k"]
        x, xs = codes[token], scale[token]
        v = [torch.matmul(x, w.float().t()) * (xs * ws) for w, ws in zip(s["w"][e], s["w_scales"][e])]
        y = v[0]
        if s["act"] == "swish":
            y = y / (1.0 + (-y).exp())
        elif s["act"] == "gelu":
            y = y / (1.0 + (y * (y * y * 0.044715 + 1.0) * (-2.0 * math.sqrt(2.0 / math.pi))).exp())
        else:
            y = y.clamp(min=0.0)
        h[a:b] = (y * v[1] if s["gated"] else y).to(h.dtype)
    return h


def _down(s):
    codes, scale = _codes(s["h"])
    y = torch.zeros(s["T"] * s["k"], s["N"], device="cuda")
    for e in range(s["E"]):
        a, b = s["starts"][e], s["starts"][e + 1]
        if a < b:
            y[s["rows"][a:b].long()] = torch.matmul(codes[a:b], s["w"][e, 0].float().t()) * (scale[a:b] * s["w_scales"][e])
    out = (y.reshape(s["T"], s["k"], -1) * s["weights"][..., None]).sum(1)
    return (out if s["residual"] is None else out + s["residual"].float()).to(s["h"].dtype)


def _adapters(s):
    out = s["base"].clone()
    r = s["R"]
    for i in range(s["A"]):
        a, b = s["starts"][i], s["starts"][i + 1]
        if a == b:
            continue
        row = s["rows"][a:b].long()
        x, at = s["x"][row].float(), 0
        kept = None if s["ranks"] is None else torch.arange(r, device="cuda") < s["ranks"][i]
        for j, n in enumerate(_slices(s)):
            v = torch.matmul(x, s["a"][i, j * r:(j + 1) * r].float().t())
            if kept is not None:
                v = torch.where(kept, v, torch.zeros((), device="cuda"))
            delta = torch.matmul(v, s["b"][i, at:at + n].float().t()) * s["scales"][i]
            out[row, at:at + n] = (s["base"][row, at:at + n].float() + delta).to(out.dtype)
            at += n
    return out


# ---------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    global own
    was, own = own, False
    s = prepare(case, seed)
    own = was
    n = case["T"]
    if case["kind"] == "route":
        return _exact_route(s)
    if case["kind"] == "adapters":
        out = s["base"].double()
        member = torch.full((n,), -1, dtype=torch.long, device="cuda")
        for i in range(case["A"]):
            member[s["rows"][s["starts"][i]:s["starts"][i + 1]].long()] = i
        column = 0
        for j, width in enumerate(_slices(case)):
            for i in member.unique().tolist():
                if i < 0:
                    continue
                rank = case["R"] if s["ranks"] is None else int(s["ranks"][i])
                here = (member == i).nonzero()[:, 0]
                left = s["a"][i].double()[j * case["R"]:j * case["R"] + rank]
                right = s["b"][i].double()[column:column + width, :rank]
                out[here, column:column + width] += (s["x"][here].double() @ left.T.contiguous()) @ right.T.contiguous() * s["scales"][i].double()
            column += width
        return out
    x = s["x"] if case["kind"] == "up" else s["h"]
    largest = x.double().abs().max(-1)[0]
    step = torch.maximum((largest / 127 * torch.ones_like(largest)).to(torch.float32), torch.full_like(largest, 2.0 ** -100).float()).double()
    whole = torch.round(x.double() / step[:, None])
    rows = s["rows"].long()
    if case["kind"] == "up":
        h = torch.zeros(n * case["k"], case["N"], dtype=torch.float64, device="cuda")
    else:
        out = torch.zeros(n, case["N"], dtype=torch.float64, device="cuda") if s["residual"] is None else s["residual"].double()
    for e in range(case["E"]):
        at = torch.arange(s["starts"][e], s["starts"][e + 1], device="cuda")
        if at.numel() == 0:
            continue
        source = rows[at] // case["k"] if case["kind"] == "up" else at
        z = [whole[source] @ (w.double() * ws.double()[:, None]).T.contiguous() * step[source, None] for w, ws in zip(s["w"][e], s["w_scales"][e])]
        if case["kind"] == "down":
            slot = rows[at]
            out.index_add_(0, slot // case["k"], z[0] * s["weights"].reshape(-1)[slot].double()[:, None])
            continue
        a = z[0]
        if case["act"] == "swish":
            a = a * torch.sigmoid(a)
        elif case["act"] == "gelu":
            a = 0.5 * a * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (a + 0.044715 * a ** 3)))
        else:
            a = torch.where(a > 0, a, torch.zeros_like(a))
        h[at] = a * z[1] if case["gated"] else a
    return h if case["kind"] == "up" else out


def _exact_route(s):
    """Each token's experts one after the other: the best that is left, the first of equals."""
    x = s["logits"].double()
    score = torch.softmax(x, -1) if s["score"] == "softmax" else torch.sigmoid(x)
    rank = score.clone()
    if s["bias_of"] is not None:
        rank += s["bias_of"].double()
    e, size = s["E"], s["E"] // s["groups"]
    if s["groups"] > 1:
        value = torch.stack([rank[:, i * size:(i + 1) * size].topk(s["best"], -1)[0].sum(-1) for i in range(s["groups"])], -1)
        open_ = torch.zeros(s["T"], s["groups"], dtype=torch.bool, device="cuda")
        for _ in range(s["top_groups"]):
            top = value.amax(-1, keepdim=True)
            first = (value == top).to(torch.int8).argmax(-1, keepdim=True)
            open_.scatter_(1, first, True)
            value.scatter_(1, first, -math.inf)
        rank[~open_.repeat_interleave(size, 1)] = -math.inf
    ids = []
    for _ in range(s["k"]):
        first = (rank == rank.amax(-1, keepdim=True)).to(torch.int8).argmax(-1, keepdim=True)
        ids.append(first)
        rank.scatter_(1, first, -math.inf)
    ids = torch.cat(ids, -1)
    w = score.gather(1, ids)
    if s["renorm"]:
        w = w / w.sum(-1, keepdim=True)
    flat = ids.reshape(-1)
    rows = torch.argsort(flat * (flat.numel() + 1) + torch.arange(flat.numel(), device="cuda"))
    counts = torch.bincount(flat, minlength=e)
    return {"experts": ids.to(torch.int32), "weights": w * s["scale"], "offsets": torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32),
            "rows": rows.to(torch.int32)}


def work(case):
    """Each input read once, each output written once, and the arithmetic of the definition."""
    n, b = case["T"], _BYTES[case["type"]]
    if case["kind"] == "route":
        return {"bytes": n * (case["E"] * b + case["k"] * 12) + case["E"] * 8 + 4, "flops": 8.0 * n * case["E"]}
    if case["kind"] == "adapters":
        out, used = sum(_slices(case)), case["A"] * (1 - (1 - 1 / case["A"]) ** min(n, 2 * case["A"] if n > 64 else n))
        deep = len(_slices(case)) * case["K"]
        return {"bytes": n * (case["K"] + 2 * out) * b + used * case["R"] * (deep + out) * b, "flops": 2.0 * n * case["R"] * (deep + out)}
    each = 2 if case["kind"] == "up" and case["gated"] else 1
    share = 0.5 if case["part"] else 1.0
    slots = n * case["k"] * share
    used = case["E"] * (1 - (1 - case["k"] * share / case["E"]) ** n)
    weights = used * each * case["N"] * (case["K"] + 4)
    rows = n * case["K"] * b + slots * case["N"] * b if case["kind"] == "up" else slots * case["K"] * b + n * case["N"] * b * (2 if case["addend"] else 1)
    return {"bytes": rows + weights, "flops": 2.0 * slots * each * case["N"] * case["K"]}
