"""The operators between a decoder's qkv linear and its output linear, as cases that can be timed and compared: norm and
rotation of queries and keys, appending to a paged cache held in 4 bits, attention over that cache.

kind        one pass
norm_rope   per-head RMS norm (where the network has one) and position rotation of the queries and keys of packed qkv rows
append      the same for rows whose keys and values go into the cache, the queries written out, and the rows read back
attention   attention of a ragged batch of new tokens over their sequences' pages, with the log-sum-exp of each row

Cache: `pages` rows of bytes. A row holds, for each kv head, K codes [P][DP / 2], V codes [P / 4][DP / 8][4][4], K parameters
and V parameters, each [P / 4][8] halves (4 scales, 4 offsets): P tokens a page, DP the head padded to 64, 128 or 256. A byte
holds two codes, the lower dimension in the low bits; value = scale * (code - 8) + offset.
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
        # queries and keys of one new token of an 8B-parameter decoder with normed heads
        dict(name="norm_rope_1", kind="norm_rope", T=1, Hq=32, Hkv=8, D=128, R=128, layout="half", norm=True, scaling="none", far=False, type="bfloat16"),
        # ... of a prompt
        dict(name="norm_rope_8192", kind="norm_rope", T=8192, Hq=32, Hkv=8, D=128, R=128, layout="half", norm=True, scaling="none", far=False, type="bfloat16"),
        # an odd number of tokens at far positions, part of a narrow head rotated, interleaved, frequencies stretched
        dict(name="norm_rope_1003_far", kind="norm_rope", T=1003, Hq=12, Hkv=12, D=80, R=32, layout="interleaved", norm=False, scaling="yarn", far=True, type="float"),
        # 64 served sequences append a token each
        dict(name="append_64", kind="append", T=64, Hq=32, Hkv=8, D=128, R=128, layout="half", norm=False, scaling="llama3", far=False, P=64, type="bfloat16"),
        # a prompt goes into the cache
        dict(name="append_8192", kind="append", T=8192, Hq=32, Hkv=8, D=128, R=128, layout="half", norm=True, scaling="none", far=False, P=64, type="bfloat16"),
        # a ragged number of rows, some of them padding that has no place in the cache, small pages
        dict(name="append_333_padded", kind="append", T=333, Hq=12, Hkv=12, D=64, R=64, layout="interleaved", norm=False, scaling="linear", far=True, P=16, type="half"),
        # one sequence's next token: latency
        dict(name="decode_1x2000", kind="attention", B=1, Q=1, L=2000, Hq=32, Hkv=8, D=128, P=16, window=0, type="bfloat16"),
        # one sequence with a long context
        dict(name="decode_1x131072", kind="attention", B=1, Q=1, L=131072, Hq=32, Hkv=8, D=128, P=64, window=0, type="bfloat16"),
        # a served batch of ragged lengths
        dict(name="decode_64x8192", kind="attention", B=64, Q=1, L=8192, Hq=32, Hkv=8, D=128, P=64, window=0, type="bfloat16"),
        # a few drafted tokens a sequence, heads of their own, in fp32
        dict(name="draft_7x1500_float", kind="attention", B=7, Q=5, L=1500, Hq=12, Hkv=12, D=64, P=32, window=0, type="float"),
        # chunks of several prompts behind what they have cached, a sliding window
        dict(name="chunk_6x500x3500", kind="attention", B=6, Q=500, L=3500, Hq=28, Hkv=4, D=128, P=32, window=1024, type="half"),
        # a whole prompt
        dict(name="prompt_8192", kind="attention", B=1, Q=8192, L=8192, Hq=32, Hkv=8, D=128, P=64, window=0, type="bfloat16"),
    ]


def _log(rng, lo, hi):
    """A size between lo and hi, even over its logarithm."""
    return max(1, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi)))))))


def draw(rng):
    kind = rng.choice(["norm_rope", "append", "decode", "draft", "prompt"])
    hkv, group = rng.choice([(8, 4), (8, 8), (4, 7), (12, 1), (2, 8), (1, 12), (5, 3)])
    d = rng.choice([64, 64, 80, 96, 128, 128, 128, 256])
    common = dict(Hq=hkv * group, Hkv=hkv, D=d)
    if kind in ("norm_rope", "append"):
        c = dict(kind=kind, T=_log(rng, 1, (8192 * 40 * 128) // ((hkv * group + 2 * hkv) * d)), **common, R=rng.choice([d, d, d // 2, 16]),
                 layout=rng.choice(["half", "interleaved"]), norm=rng.choice([True, False]),
                 scaling=rng.choice(["none", "linear", "llama3", "yarn"]), far=rng.choice([True, False]))
        if kind == "append":
            c["P"] = rng.choice([16, 32, 64, 128])
        return dict(c, type=rng.choice(["bfloat16", "half", "float"]))
    common.update(P=rng.choice([16, 32, 64, 128]), window=rng.choice([0, 0, 0, 128, 1000]))
    if kind == "decode":
        b = _log(rng, 1, 64)
        longest = min(131072, (64 * 8192 * 8 * 128) // (b * hkv * 2 * max(64, d)))
        return dict(kind="attention", B=b, Q=1, L=_log(rng, 16, longest), **common, type=rng.choice(["bfloat16", "half"]))
    if kind == "draft":
        b, q = _log(rng, 1, 32), rng.randint(2, 16)
        longest = min(16384, (1 << 25) // (b * q * hkv * group))
        return dict(kind="attention", B=b, Q=q, L=q + _log(rng, 16, longest), **common, type=rng.choice(["bfloat16", "half", "float"]))
    t = rng.choice(["bfloat16", "half", "half", "bfloat16", "float"])
    b, q = _log(rng, 1, 8), _log(rng, 32, 2048 if t != "float" else 500)
    longest = min(8192, (1 << 37) // (b * q * hkv * group * max(d, 128)))
    return dict(kind="attention", B=b, Q=q, L=max(q, _log(rng, 32, max(32, longest))), **common, type=t)


# ---------------------------------------------------------------------------------------------------------------------
# what a program has in hand before the call
# ---------------------------------------------------------------------------------------------------------------------
def _frequencies(r, scaling):
    """(turns a position for each rotated pair, in 64 bits; the factor on cosine and sine)"""
    if scaling == "linear":      # positions compressed by 4
        return 10000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64) / r) / (2 * math.pi) / 4.0, 1.0
    if scaling == "llama3":      # base 500000; long wavelengths compressed by 8, a ramp between 2048 and 8192 positions
        f = 500000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64) / r) / (2 * math.pi)
        ramp = ((8192.0 * f - 1.0) / (4.0 - 1.0)).clamp(0.0, 1.0)
        return f * ramp + f / 8.0 * (1.0 - ramp), 1.0
    if scaling == "yarn":        # 16 times the trained 4096 positions; pairs of 1 to 32 turns in them on a linear ramp
        f = 10000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64) / r) / (2 * math.pi)
        at = [r * math.log(4096.0 / (turns * 2 * math.pi)) / (2 * math.log(10000.0)) for turns in (32.0, 1.0)]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), r - 1)
        ramp = ((torch.arange(r // 2, dtype=torch.float64) - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
        return f / 16.0 * ramp + f * (1.0 - ramp), 0.1 * math.log(16.0) + 1.0
    return 500000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64) / r) / (2 * math.pi), 1.0


def _padded(d):
    return 64 if d <= 64 else 128 if d <= 128 else 256


def _random_pages(case, pages, g):
    """A cache in use: codes and parameters of roughly normal keys and values."""
    h, p, dp = case["Hkv"], case["P"], _padded(case["D"])
    n = pages * h

    def codes():
        c = torch.empty(n, p * dp, device="cuda").normal_(generator=g).mul_(2.6).sub_(0.5).round_().clamp_(-8, 7).add_(8).to(torch.uint8)
        return c[:, 0::2] | (c[:, 1::2] << 4)

    def parameters(scale, spread):
        s = (torch.randn(n, p // 4, 4, device="cuda", generator=g) * 0.15).exp_() * scale
        o = torch.randn(n, p // 4, 4, device="cuda", generator=g) * spread + 0.5 * s
        return torch.cat([s, o], -1).to(torch.float16).reshape(n, p * 2).view(torch.uint8)

    return torch.cat([codes(), codes(), parameters(0.36, 0.1), parameters(0.36, 0.1)], 1).reshape(pages, -1)


def _lengths(case):
    """(new tokens, tokens in the cache with them) of each sequence: the first has the full sizes, the others are ragged."""
    rng = random.Random(case["B"] * 1000003 + case["Q"] * 1009 + case["L"])
    new = [case["Q"]] + [rng.randint(1, case["Q"]) for _ in range(case["B"] - 1)]
    return new, [max(n, case["L"] if i == 0 else rng.randint(max(1, case["L"] // 4), case["L"])) for i, n in enumerate(new)]


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = dict(case)
    hq, hkv, d, t = case["Hq"], case["Hkv"], case["D"], _TORCH[case["type"]]
    if case["kind"] in ("norm_rope", "append"):
        n = case["T"]
        spread = (torch.randn(1, hq + 2 * hkv, d, device="cuda", generator=g) * 0.25).exp_()   # channels differ in size
        s["qkv"] = (torch.randn(n, hq + 2 * hkv, d, device="cuda", generator=g) * spread).to(t)   # the qkv linear's output
        s["q"], s["k"], s["v"] = s["qkv"][:, :hq], s["qkv"][:, hq:hq + hkv], s["qkv"][:, hq + hkv:]
        freqs, s["factor"] = _frequencies(case["R"], case["scaling"])
        s["freqs"] = freqs.cuda()
        start = torch.randint(0, 900000 if case["far"] else 4096, (1,), device="cuda", generator=g)
        s["positions"] = (start + torch.arange(n, device="cuda")).to(torch.int32)
        s["wq"], s["wk"] = ((1.0 + 0.2 * torch.randn(d, device="cuda", generator=g)) if case["norm"] else None for _ in range(2))
        s["q_out"], s["k_out"] = torch.empty(n, hq, d, dtype=t, device="cuda"), torch.empty(n, hkv, d, dtype=t, device="cuda")
        if case["kind"] == "append":
            s["pages"] = -(-n // case["P"]) + 3
            where = torch.randperm(s["pages"], device="cuda", generator=g)
            row = torch.arange(n, device="cuda")
            s["slots"] = where[row // case["P"]] * case["P"] + row % case["P"]
            if n > 100 and n % 2:
                s["slots"][::10] = -1    # padded rows
            s["cache"] = torch.zeros(s["pages"], hkv * case["P"] * (_padded(d) + 8), dtype=torch.uint8, device="cuda")
            s["v_out"] = torch.empty_like(s["k_out"])
    else:
        b, q, longest, p = case["B"], case["Q"], case["L"], case["P"]
        new, length = (torch.tensor(v, device="cuda") for v in _lengths(case))
        s["kv_len"] = length.to(torch.int32)
        s["cu_q"] = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), new.cumsum(0)]).to(torch.int32)
        s["rows"] = int(s["cu_q"][-1])
        width = -(-longest // p)
        used = (length + p - 1) // p
        s["pages"] = int(used.sum()) + 2
        where = torch.randperm(s["pages"], device="cuda", generator=g)
        column = torch.arange(width, device="cuda")
        at = used.cumsum(0)[:, None] - used[:, None] + column[None, :]
        s["table"] = torch.where(column[None, :] < used[:, None], where[at.clamp(max=s["pages"] - 1)], -1).to(torch.int32)
        s["cache"] = _random_pages(case, s["pages"], g)
        s["query"] = (torch.randn(s["rows"], hq, d, device="cuda", generator=g) * 1.3).to(t)
        s["out"] = torch.empty(s["rows"], hq, d, dtype=t, device="cuda")
        s["lse"] = torch.empty(s["rows"], hq, dtype=torch.float32, device="cuda")
    if own:
        _plan(s)
    return s


def _plan(s):
    """What a program that calls the framework keeps: its parameter structures and workspace."""
    hip = importlib.import_module("intel-extension-for-tensorflow_amd").itexhip
    t = {"float": hip.FLOAT, "bfloat16": hip.BFLOAT16, "half": hip.HALF}[s["type"]]
    s["hip"], s["t"] = hip, t
    if s["kind"] != "norm_rope":
        s["geometry"] = hip.kv4_cache(s["D"], s["Hkv"], s["P"], s["pages"])
    if s["kind"] == "attention":
        s["params"] = hip.kv4_attention_params(t, s["Hq"], s["D"], s["B"], s["Q"], s["rows"], s["D"] ** -0.5, table_stride=s["table"].shape[1],
                                               window=s["window"])
        s["workspace"] = torch.empty(hip.kv4_attention_workspace(s["params"], s["geometry"]), dtype=torch.uint8, device="cuda")
    else:
        row = (s["qkv"].stride(0), s["qkv"].stride(1))
        s["params"] = hip.heads_params(t, s["D"], s["Hq"], s["Hkv"], rotary_dim=s["R"], interleaved=s["layout"] == "interleaved", eps=1e-6,
                                       attention_factor=s["factor"], q_strides=row, k_strides=row, v_strides=row)


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(s):
    if own:
        return _run_own(s)
    if s["kind"] == "attention":
        return _attend(s)
    q = _norm_rotate(s, s["q"], s["wq"])
    k = _norm_rotate(s, s["k"], s["wk"])
    if s["kind"] == "norm_rope":
        return {"q": q.to(s["qkv"].dtype), "k": k.to(s["qkv"].dtype)}
    kept = (s["slots"] >= 0)[:, None, None]
    return {"q": q.to(s["qkv"].dtype), "k": _through_4_bits(k, kept).to(s["qkv"].dtype), "v": _through_4_bits(s["v"].double(), kept).to(s["qkv"].dtype)}


def _run_own(s):
    hip = s["hip"]
    if s["kind"] == "attention":
        hip.kv4_attention(s["params"], s["geometry"], s["query"], s["cache"], s["table"], s["cu_q"], s["kv_len"], s["workspace"], s["out"], s["lse"])
        return {"out": s["out"], "lse": s["lse"]}
    if s["kind"] == "norm_rope":
        hip.qk_norm_rope(s["params"], s["T"], s["q"], s["k"], s["wq"], s["wk"], s["positions"], s["freqs"], s["q_out"], s["k_out"])
        return {"q": s["q_out"], "k": s["k_out"]}
    hip.kv4_append(s["params"], s["geometry"], s["T"], s["q"], s["k"], s["v"], s["wq"], s["wk"], s["positions"], s["freqs"], s["slots"],
                   s["q_out"], s["cache"])
    hip.kv4_gather(s["geometry"], s["t"], s["T"], s["cache"], s["slots"], s["k_out"], s["v_out"])
    return {"q": s["q_out"], "k": s["k_out"], "v": s["v_out"]}


def _norm_rotate(s, x, w):
    """In 64 bits where codes follow (values next to a border), in 32 otherwise; the angles in 64."""
    x = x.double() if s["kind"] == "append" else x.float()
    if w is not None:
        x = x * (x.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w.to(x.dtype)
    turns = s["positions"].double()[:, None] * s["freqs"]
    angle = (turns - turns.floor()) * (2 * math.pi)
    c, z = ((f * s["factor"]).to(x.dtype)[:, None, :] for f in (angle.cos(), angle.sin()))
    r = s["R"]
    if s["layout"] == "half":
        a, b = x[..., :r // 2], x[..., r // 2:r]
        return torch.cat([a * c - b * z, b * c + a * z, x[..., r:]], -1)
    a, b = x[..., 0:r:2], x[..., 1:r:2]
    return torch.cat([torch.stack([a * c - b * z, b * c + a * z], -1).flatten(-2), x[..., r:]], -1)


def _through_4_bits(x, kept):
    """The values that the cache stands for; zero for rows that have no place in it."""
    x = x.clamp(-65504.0, 65504.0)
    hi, lo = x.amax(-1, keepdim=True), x.amin(-1, keepdim=True)
    scale = ((hi - lo) / 15.0).half().double()
    offset = (lo + 8.0 * scale).half().double()
    code = torch.where(scale > 0, ((x - offset) / scale).round(), torch.zeros_like(x)).clamp(-8.0, 7.0)
    return torch.where(kept, scale * code + offset, torch.zeros_like(x))


def _values(s):
    """Keys and values of every sequence [B, Hkv, W P, D] from its pages, in 32 bits."""
    b, width = s["table"].shape
    h, p, dp = s["Hkv"], s["P"], _padded(s["D"])
    block = s["cache"][s["table"].clamp(min=0).long().reshape(-1)].reshape(b, width, h, -1)
    k, v, kp, vp = block.split([p * dp // 2, p * dp // 2, p * 4, p * 4], -1)
    v = v.reshape(b, width, h, p // 4, dp // 8, 4, 4).transpose(4, 5).reshape(b, width, h, p * dp // 2)

    def dequantized(codes, params):
        codes = torch.stack([codes & 15, codes >> 4], -1).reshape(b, width, h, p, dp)[..., :s["D"]].float() - 8.0
        params = params.contiguous().view(torch.float16).reshape(b, width, h, p // 4, 2, 4).float()
        scale, offset = params[..., 0, :].reshape(b, width, h, p, 1), params[..., 1, :].reshape(b, width, h, p, 1)
        return (codes * scale + offset).transpose(1, 2).reshape(b, h, width * p, s["D"])

    return dequantized(k, kp), dequantized(v, vp)


def _attend(s):
    b, d, hq, hkv = s["B"], s["D"], s["Hq"], s["Hkv"]
    group, most = hq // hkv, s["Q"]
    k, v = _values(s)
    n = k.shape[2]
    first = s["cu_q"][:-1].long()
    count = s["cu_q"][1:].long() - first
    i = torch.arange(most, device=k.device)
    row = (first[:, None] + i).clamp(max=s["rows"] - 1)                                  # [B, Q]
    q = s["query"].float()[row].reshape(b, most, hkv, group, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, group * most, d)
    scores = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(d ** -0.5).reshape(b, hkv, group, most, n)
    at = s["kv_len"].long()[:, None] - count[:, None] + i                                # position of each new token
    t = torch.arange(n, device=k.device)
    seen = (t <= at[..., None]) & (i < count[:, None])[..., None]
    if s["window"]:
        seen = seen & (t > at[..., None] - s["window"])
    seen = seen[:, None, None]
    scores.masked_fill_(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    v = torch.where((t < s["kv_len"].long()[:, None])[:, None, :, None], v, torch.zeros((), device=v.device))
    out = torch.matmul(p.reshape(b, hkv, group * most, n), v).reshape(b, hkv, group, most, d) / total.clamp(min=1e-30)
    lse = (total.log() + top)[..., 0]
    keep = (i < count[:, None]).reshape(-1)
    out = out.permute(0, 3, 1, 2, 4).reshape(b * most, hq, d)[keep]
    return {"out": out.to(s["query"].dtype), "lse": lse.permute(0, 3, 1, 2).reshape(b * most, hq)[keep]}


# ---------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits, a head or a sequence at a time
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    global own
    was, own = own, False
    s = prepare(case, seed)
    own = was
    if case["kind"] == "attention":
        return _exact_attention(s)
    r, half = case["R"], case["R"] // 2
    phase = torch.outer(s["positions"].double(), s["freqs"]).fmod(1.0) * (2 * math.pi)
    turn = torch.polar(torch.full_like(phase, s["factor"]), phase)[:, None, :]

    def rotated(x, w):
        x = x.double()
        if w is not None:
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / case["D"] + 1e-6) * w.double()
        x = x.clone()
        pair = (slice(0, half), slice(half, r)) if case["layout"] == "half" else (slice(0, r, 2), slice(1, r, 2))
        z = torch.complex(x[..., pair[0]].contiguous(), x[..., pair[1]].contiguous()) * turn
        x[..., pair[0]], x[..., pair[1]] = z.real, z.imag
        return x

    q, k = rotated(s["q"], s["wq"]), rotated(s["k"], s["wk"])
    if case["kind"] == "norm_rope":
        return {"q": q, "k": k}

    def cached(x):
        top, bottom = x.max(-1, keepdim=True)[0], x.min(-1, keepdim=True)[0]
        step = ((top - bottom) / 15).to(torch.float16).double()
        centre = (bottom + step * 8).to(torch.float16).double()
        steps = torch.round((x - centre) / torch.where(step == 0, torch.ones_like(step), step)).clamp(-8, 7)
        x = centre + steps * step
        x[s["slots"] < 0] = 0
        return x

    return {"q": q, "k": cached(k), "v": cached(s["v"].double())}


def _exact_attention(s):
    p, dp, d, hkv, hq = s["P"], _padded(s["D"]), s["D"], s["Hkv"], s["Hq"]
    codes = p * dp // 2
    out = torch.zeros(s["rows"], hq, d, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["rows"], hq, dtype=torch.float64, device="cuda")
    cu, lengths = s["cu_q"].tolist(), s["kv_len"].tolist()

    def nibbles(x):
        return torch.stack([x.remainder(16), x.div(16, rounding_mode="floor")], -1).flatten(-2).double() - 8

    for b, n in enumerate(lengths):
        pages = s["table"][b, :-(-n // p)].long()
        rows = slice(cu[b], cu[b + 1])
        m = cu[b + 1] - cu[b]
        at = torch.arange(n - m, n, device="cuda")[:, None]
        t = torch.arange(n, device="cuda")[None, :]
        hidden = (t > at) | ((t <= at - s["window"]) if s["window"] else (t < 0))
        for h in range(hkv):
            size = p * (dp + 8)
            block = s["cache"][pages, h * size:(h + 1) * size]
            kq = nibbles(block[:, :codes].reshape(-1, dp // 2))[:n, :d]
            vq = nibbles(block[:, codes:2 * codes].reshape(-1, dp // 8, 4, 4).permute(0, 2, 1, 3).reshape(-1, dp // 2))[:n, :d]
            kp, vp = (block[:, c:c + 4 * p].contiguous().view(torch.float16).reshape(-1, 2, 4).double() for c in (2 * codes, 2 * codes + 4 * p))
            k = kq * kp[:, 0].reshape(-1, 1)[:n] + kp[:, 1].reshape(-1, 1)[:n]
            v = vq * vp[:, 0].reshape(-1, 1)[:n] + vp[:, 1].reshape(-1, 1)[:n]
            for j in range(hq // hkv):
                head = h * (hq // hkv) + j
                z = (s["query"][rows, head].double() @ k.T.contiguous()) / math.sqrt(d)
                z[hidden] = -math.inf
                lse[rows, head] = z.logsumexp(-1)
                out[rows, head] = torch.exp(z - lse[rows, head][:, None]) @ v
    return {"out": out, "lse": lse}


def work(case):
    """Each input read once, each output written once, and the arithmetic of the definition."""
    hq, hkv, d, e = case["Hq"], case["Hkv"], case["D"], _BYTES[case["type"]]
    row = hkv * (_padded(d) + 8)
    if case["kind"] == "attention":
        w, pairs, read, new = case["window"] or case["L"], 0, 0, 0
        for q, n in zip(*_lengths(case)):
            pairs += sum(min(w, n - i) for i in range(q))
            read += min(n, w + q - 1)
            new += q
        return {"bytes": read * row + new * hq * (2 * d * e + 4), "flops": 4.0 * pairs * hq * d}
    n = case["T"]
    if case["kind"] == "norm_rope":
        return {"bytes": n * (2 * (hq + hkv) * d * e + 4), "flops": 8.0 * n * (hq + hkv) * d}
    return {"bytes": n * ((2 * hq + 2 * hkv) * d * e + 2 * row + 2 * hkv * d * e + 12), "flops": 12.0 * n * (hq + 2 * hkv) * d}
