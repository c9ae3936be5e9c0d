"""The experts' products, against their statement in 64 bits.

Exact where it can be: rows whose largest value is 127 have a scale of 1, whole numbers are their own codes, scales are powers of two and sums stay
below 2^24, so that a result is one rounding of a whole number.  Elsewhere a value v = fp32(sum) * (s * scale) has three roundings, 3 2^-24 |v|; an
activation y of it follows with its slope (at most 1.13) and its own evaluation: swish and the tanh gelu through exp2 of an argument a within
a few steps of |a| and a reciprocal, (16 + 8 |a|) 2^-24 |y|, the erf gelu 1e-6 + 2e-6 |y|; the product with v1 adds 4 steps; a weighted sum of k
choices and an addend adds k + 2 steps of the sum of their sizes; each result is then rounded to its type, eps / 2."""
import math

import pytest
import torch

from tests import chosen_reference as ref

pytestmark = pytest.mark.gpu
STEP = 2.0 ** -24


def type_of(hip, name):
    return {"float": hip.FLOAT, "bfloat16": hip.BFLOAT16, "half": hip.HALF}[name]


def act_of(hip, name):
    return {"none": hip.ACT_NONE, "relu": hip.ACT_RELU, "gelu_approx": hip.ACT_GELU_APPROX, "gelu_exact": hip.ACT_GELU_EXACT, "swish": hip.ACT_SWISH}[name]


def pack(hip, dev, w):
    e, each, n, k = w.shape
    packed = torch.empty(e, each, hip.qgemm_packed_bytes(k, n), dtype=torch.int8, device=dev)
    sums = torch.empty(n, dtype=torch.int32, device=dev)
    wd = w.to(dev)
    for i in range(e):
        for j in range(each):
            hip.qgemm_prepack_b(wd[i, j], True, k, n, packed[i, j], sums)
    torch.cuda.synchronize()
    return packed


def guarded(n, dev):
    """Device bytes with a border that a call must leave"""
    return torch.full((n + 256,), 0x5a, dtype=torch.uint8, device=dev)


def run_up(hip, dev, name, x, offsets, rows, top_k, w, scales, activation, gated, packed=None, stream=0, x_stride=None):
    t, k = x.shape
    p = hip.experts_params(type_of(hip, name), w.shape[0], top_k, t, k, w.shape[2], activation=act_of(hip, activation), gated=gated, x_stride=x_stride)
    xd = x.to(dev)
    if x_stride is not None:
        wide = torch.full((t, x_stride), 1000.0, dtype=x.dtype, device=dev)
        wide[:, :k] = xd
        xd = wide
    packed = pack(hip, dev, w) if packed is None else packed
    h = torch.full((t * top_k + 1, w.shape[2]), 7.0, dtype=x.dtype, device=dev)
    size = hip.experts_workspace(p)
    work = guarded(size, dev)
    hip.experts_up(p, xd, offsets.to(dev), rows.to(dev), packed, scales.to(dev), h, work, stream)
    torch.cuda.synchronize()
    assert bool((work[size:] == 0x5a).all())
    last = int(offsets[-1])
    assert bool((h[last:] == 7).all())          # rows behind the last group are left
    return h[:-1].cpu()


def run_down(hip, dev, name, h, experts, offsets, rows, w, scales, weights, addend, packed=None, in_place=False, stride=None):
    t, top_k = experts.shape
    k, n = h.shape[1], w.shape[2]
    p = hip.experts_params(type_of(hip, name), w.shape[0], top_k, t, n, k, activation=hip.ACT_NONE, gated=False, addend_stride=stride, out_stride=stride)
    packed = pack(hip, dev, w) if packed is None else packed
    out = torch.full((t, stride or n), 7.0, dtype=h.dtype, device=dev)
    ad = None
    if addend is not None:
        ad = out if in_place else torch.full_like(out, 9.0)
        ad[:, :n] = addend.to(dev)
    size = hip.experts_workspace(p)
    work = guarded(size, dev)
    hip.experts_down(p, h.to(dev), experts.to(dev), offsets.to(dev), rows.to(dev), packed, scales.to(dev), weights.to(dev), ad, out, work)
    torch.cuda.synchronize()
    assert bool((work[size:] == 0x5a).all()) and bool((out[:, n:] == 7).all())
    return out[:, :n].cpu()


def choices(t, k, e, seed, total=None, skew=0.0):
    g = torch.Generator().manual_seed(seed)
    score = torch.rand(t, total or e, generator=g) + skew * torch.linspace(1, 0, total or e)
    return score.topk(k, -1)[1].to(torch.int32)


def whole(shape, limit, g, largest=None):
    x = torch.randint(-limit, limit + 1, shape, generator=g).float()
    if largest is not None:
        at = torch.randint(0, shape[-1], shape[:-1] + (1,), generator=g)
        x.scatter_(-1, at, largest)
    return x


SIZES = [  # tokens, top_k, experts, K, N, total experts
    (1, 2, 8, 64, 32, 8), (1, 1, 1, 1, 1, 1), (2, 2, 4, 33, 31, 4), (5, 3, 7, 100, 65, 14), (33, 4, 6, 200, 130, 6), (64, 6, 64, 256, 96, 64), (31, 1, 3, 1000, 40, 3),
    (300, 2, 4, 128, 264, 8), (129, 8, 16, 72, 48, 16), (700, 2, 3, 64, 70, 3), (3, 32, 40, 64, 33, 80), (40, 1, 1024, 48, 32, 1024), (600, 1, 1, 192, 512, 1), (1100, 4, 5, 320, 136, 5),
    (1, 32, 40, 64, 33, 80), (2, 16, 20, 80, 40, 20), (4, 8, 64, 100, 64, 64), (16, 2, 5, 64, 100, 5), (8, 3, 3, 1000, 33, 6), (2, 1, 2, 8192, 40, 2), (13, 1, 1, 512, 96, 1),
    (1500, 2, 3, 256, 600, 3), (3200, 2, 16, 200, 2100, 16), (1030, 2, 4, 449, 1100, 8), (4, 2, 2, 14336, 70, 2)]


@pytest.mark.parametrize("name", list(ref.TYPES))
@pytest.mark.parametrize("t,k,e,K,N,total", SIZES)
def test_up_exactly(hip, dev, name, t, k, e, K, N, total):
    g = torch.Generator().manual_seed(t + K)
    x = whole((t, K), 3, g, largest=127.0).to(ref.TYPES[name])
    w = whole((e, 2, N, K), 4, g).to(torch.int8)
    scales = 2.0 ** torch.randint(-7, -3, (e, 2, N), generator=g).float()
    offsets, rows = ref.order(choices(t, k, e, 7 * t + e, total), e)
    packed = pack(hip, dev, w)
    for gated in (True, False):
        # (a gated result may have more bits than fp32: one more rounding before the type's)
        want = ref.up(x, offsets, rows, k, w[:, :1 + gated], scales[:, :1 + gated], "none", gated)[:int(offsets[-1])]
        got = run_up(hip, dev, name, x, offsets, rows, k, w[:, :1 + gated], scales[:, :1 + gated].contiguous(), "none", gated,
                     packed[:, :1 + gated].contiguous())[:int(offsets[-1])]
        assert torch.equal(got, want.float().to(got.dtype)), (gated, (got.double() - want).abs().max())


@pytest.mark.parametrize("name", list(ref.TYPES))
@pytest.mark.parametrize("t,k,e,K,N,total", SIZES)
def test_down_exactly(hip, dev, name, t, k, e, K, N, total):
    g = torch.Generator().manual_seed(t + K)
    h = whole((t * k, K), 3, g, largest=127.0).to(ref.TYPES[name])
    w = whole((e, 1, N, K), 4, g).to(torch.int8)
    scales = torch.full((e, 1, N), 0.25)
    weights = torch.randint(0, 5, (t, k), generator=g).float()
    experts = choices(t, k, e, 7 * t + e, total)
    offsets, rows = ref.order(experts, e)
    addend = whole((t, N), 100, g).to(ref.TYPES[name])
    packed = pack(hip, dev, w)
    for ad in (addend, None):
        want, _ = ref.down(h, experts, offsets, rows, w, scales, weights, ad)
        assert float(want.abs().max()) * 4 < 2 ** 24
        got = run_down(hip, dev, name, h, experts, offsets, rows, w, scales, weights, ad, packed)
        assert torch.equal(got, want.float().to(got.dtype)), (got.double() - want).abs().max()
    again = run_down(hip, dev, name, h, experts, offsets, rows, w, scales, weights, addend, packed, in_place=True, stride=N + 5)
    want, _ = ref.down(h, experts, offsets, rows, w, scales, weights, addend)
    assert torch.equal(again, want.float().to(again.dtype))


@pytest.mark.parametrize("name", list(ref.TYPES))
@pytest.mark.parametrize("activation", ["swish", "gelu_approx", "gelu_exact", "relu", "none"])
@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("t", [9, 400])
def test_up(hip, dev, name, activation, gated, t):
    k, e, K, N = 2, 5, 530, 150
    g = torch.Generator().manual_seed(t)
    x = (torch.randn(t, K, generator=g) * (torch.randn(1, K, generator=g) * 0.5).exp()).to(ref.TYPES[name])
    w = (torch.randn(e, 2, N, K, generator=g) * 33).round().clamp(-127, 127).to(torch.int8)[:, :1 + gated].contiguous()
    scales = (0.8 + 0.4 * torch.rand(e, 1 + gated, N, generator=g)) * (0.05 / K ** 0.5)
    offsets, rows = ref.order(choices(t, k, e, t), e)
    got = run_up(hip, dev, name, x, offsets, rows, k, w, scales, activation, gated, x_stride=K + 3).double()
    v0 = ref.up(x, offsets, rows, k, w[:, :1], scales[:, :1], "none", False)
    v1 = ref.up(x, offsets, rows, k, w[:, -1:], scales[:, -1:], "none", False) if gated else torch.ones_like(v0)
    y = ref.activate(activation, v0)
    a = {"swish": v0.abs(), "gelu_approx": 1.6 * v0.abs() * (1 + 0.045 * v0 ** 2)}.get(activation, torch.zeros_like(v0))
    own = 1e-6 + 2e-6 * y.abs() if activation == "gelu_exact" else (16 + 8 * a) * STEP * y.abs() if activation in ("swish", "gelu_approx") else 0.0 * y
    dy = 1.13 * 3 * STEP * v0.abs() + own
    want = y * v1
    tol = dy * v1.abs() + 4 * STEP * want.abs() + torch.finfo(ref.TYPES[name]).eps / 2 * want.abs() * (1 + 2.0 ** -10) + torch.finfo(ref.TYPES[name]).tiny * 2.0 ** -10
    off = (got - want).abs() - tol
    assert bool((off <= 0).all()), float(off.max())


@pytest.mark.parametrize("name", list(ref.TYPES))
@pytest.mark.parametrize("t,k,e,K,N", [(1, 2, 8, 1440, 516), (7, 4, 12, 1000, 770), (500, 2, 4, 300, 258)])
def test_down(hip, dev, name, t, k, e, K, N):
    g = torch.Generator().manual_seed(t)
    h = (torch.randn(t * k, K, generator=g) * torch.randn(t * k, 1, generator=g).exp()).to(ref.TYPES[name])
    w = (torch.randn(e, 1, N, K, generator=g) * 33).round().clamp(-127, 127).to(torch.int8)
    scales = (0.8 + 0.4 * torch.rand(e, 1, N, generator=g)) * (0.03 / K ** 0.5)
    weights = torch.softmax(torch.randn(t, k, generator=g), -1)
    experts = choices(t, k, e, t)
    offsets, rows = ref.order(experts, e)
    addend = torch.randn(t, N, generator=g).to(ref.TYPES[name])
    got = run_down(hip, dev, name, h, experts, offsets, rows, w, scales, weights, addend).double()
    want, size = ref.down(h, experts, offsets, rows, w, scales, weights, addend)
    tol = (4 + k + 2) * STEP * size + torch.finfo(ref.TYPES[name]).eps / 2 * want.abs() * (1 + 2.0 ** -10) + torch.finfo(ref.TYPES[name]).tiny * 2.0 ** -10
    off = (got - want).abs() - tol
    assert bool((off <= 0).all()), float(off.max())


@pytest.mark.parametrize("name", list(ref.TYPES))
def test_codes(hip, dev, name):
    """Weights that pick one element each show the codes: quotients next to halves, at them, tiny and large rows, zeros."""
    K, dtype = 64, ref.TYPES[name]
    g = torch.Generator().manual_seed(3)
    x = torch.randn(600, K, generator=g)
    x[1] = 0.0
    x[2] *= 1e-6
    x[3] *= 3e4 / x[3].abs().max()
    x[4, :] = torch.arange(K) + 0.5
    x[4, 0] = 127.0                        # scale 1: halves to even
    x[5] = x[4] * 2.0 ** -9
    if name != "half":
        x[6] *= 1e-30
        x[7] *= 1e36
        x[8] *= 1e-37
    for i in range(9, 600):                 # next to halves of the row's own scale
        s = x[i].abs().max() / 127.0
        x[i, :-1] = torch.where(x[i, :-1].abs() == x[i].abs().max(), x[i, :-1], ((x[i, :-1] / s).round() + 0.5 - 1.0 * (torch.arange(K - 1) % 2)) * s)
    x = x.to(dtype)
    w = torch.eye(K, dtype=torch.int8).reshape(1, 1, K, K)
    offsets, rows = torch.tensor([0, 600], dtype=torch.int32), torch.arange(600, dtype=torch.int32)
    codes, s = ref.quantize(x)
    scale = torch.full((1, 1, K), 2.0)
    fine = ((codes * s * 2).abs() < torch.finfo(dtype).max).all(-1)
    got = run_up(hip, dev, name, x, offsets, rows, 1, w, scale, "none", False)
    want = (codes.float() * (s.float() * 2.0)).to(dtype)
    assert torch.equal(got[fine], want[fine])


def test_rows_that_are_not_finite(hip, dev):
    t, K, N = 6, 40, 36
    x = torch.ones(t, K)
    x[1, 39], x[2, 0], x[3, 7] = math.nan, math.inf, -math.inf
    w = torch.ones(2, 1, N, K, dtype=torch.int8)
    experts = torch.tensor([[0, 1]] * t, dtype=torch.int32)
    offsets, rows = ref.order(experts, 2)
    h = run_up(hip, dev, "float", x, offsets, rows, 2, w, torch.ones(2, 1, N), "none", False)
    bad = torch.isin(rows // 2, torch.tensor([1, 2, 3]))
    assert bool(h[bad].isnan().all()) and bool(h[~bad].isfinite().all())
    # the way back: a choice that is on another device does not reach its token, whatever its weight and the row behind the last group hold
    experts[:, 1] = 5
    offsets, rows = ref.order(experts, 2)
    hh = torch.ones(2 * t, K)
    hh[int(offsets[-1]):] = math.nan
    hh[2, 3] = math.nan
    weights = torch.full((t, 2), 0.5)
    weights[:, 1] = math.nan
    out = run_down(hip, dev, "float", hh, experts, offsets, rows, w, torch.ones(2, 1, N), weights, None)
    assert bool(out[2].isnan().all()) and bool(out[[0, 1, 3, 4, 5]].isfinite().all())
    experts[4] = -1                        # a token with no expert here
    offsets, rows = ref.order(experts, 2)
    out = run_down(hip, dev, "float", torch.ones(2 * t, K), experts, offsets, rows, w, torch.ones(2, 1, N), weights, None)
    assert bool((out[4] == 0).all())


def test_orders_that_are_none_stay_inside(hip, dev):
    """Offsets and rows that are no order give no defined result, but nothing outside the outputs is read or written."""
    t, k, e, K, N = 9, 2, 3, 64, 64
    w = torch.ones(e, 1, N, K, dtype=torch.int8)
    for offsets in ([0, 5, 100, 18], [-4, 7, 3, 1 << 30], [18, 18, 18, 18], [0, 18, 0, 18], [18, 0, 18, 0]):
        offsets = torch.tensor(offsets, dtype=torch.int32)
        rows = torch.tensor([0, 17, 18, -1, 1 << 30] + [3] * 13, dtype=torch.int32)
        p = hip.experts_params(hip.FLOAT, e, k, t, K, N, activation=hip.ACT_NONE, gated=False)
        h, out = torch.zeros(t * k + 1, N, device=dev), torch.zeros(t + 1, N, device=dev)
        work = guarded(hip.experts_workspace(p), dev)
        ids = torch.zeros(t, k, dtype=torch.int32, device=dev)
        packed, ones = pack(hip, dev, w), torch.ones(e, N, device=dev)
        hip.experts_up(p, torch.ones(t, K, device=dev), offsets.to(dev), rows.to(dev), packed, ones, h, work)
        hip.experts_down(p, torch.ones(t * k, K, device=dev), ids, offsets.to(dev), rows.to(dev), packed, ones, torch.ones(t, k, device=dev), None, out, work)
        torch.cuda.synchronize()
        assert bool((h[-1] == 0).all()) and bool((out[-1] == 0).all()) and bool((work[-256:] == 0x5a).all())


def test_orders_that_are_none_stay_inside_tiles(hip, dev):
    """The same for sizes whose rows go through tiles."""
    t, k, e, K, N = 1500, 2, 3, 256, 600
    n = t * k
    w = torch.ones(e, 2, N, K, dtype=torch.int8)
    packed, ones = pack(hip, dev, w), torch.ones(e, 2, N, device=dev)
    p = hip.experts_params(hip.HALF, e, k, t, K, N, activation=hip.ACT_NONE)
    for offsets in ([0, n, 0, n], [5, 7, 1 << 30, -3], [n, 0, n, 0]):
        rows = torch.full((n,), -9, dtype=torch.int32)
        rows[::3] = 1 << 30
        h = torch.zeros(n + 1, N, dtype=torch.float16, device=dev)
        size = hip.experts_workspace(p)
        work = guarded(size, dev)
        hip.experts_up(p, torch.ones(t, K, dtype=torch.float16, device=dev), torch.tensor(offsets, dtype=torch.int32, device=dev), rows.to(dev), packed, ones, h, work)
        torch.cuda.synchronize()
        assert bool((h[-1] == 0).all()) and bool((work[size:] == 0x5a).all())


def test_a_token_that_names_an_expert_twice(hip, dev):
    """Each choice is a row of its own, also where workgroups make the codes of as many rows as there are tokens."""
    g = torch.Generator().manual_seed(8)
    for t, k, e, K, N in ((1, 2, 4, 64, 40), (3, 4, 2, 100, 40), (5, 6, 3, 64, 64), (40, 2, 2, 64, 33)):
        experts = torch.randint(0, e, (t, k), generator=g, dtype=torch.int32)
        experts[0] = 1
        offsets, rows = ref.order(experts, e)
        x, w, scales = whole((t, K), 3, g, largest=127.0), whole((e, 1, N, K), 4, g).to(torch.int8), torch.full((e, 1, N), 0.5)
        h = run_up(hip, dev, "float", x, offsets, rows, k, w, scales, "none", False)
        assert torch.equal(h, ref.up(x, offsets, rows, k, w, scales, "none", False).float())
        hh, w2, s2 = whole((t * k, N), 3, g, largest=127.0), whole((e, 1, K, N), 4, g).to(torch.int8), torch.full((e, 1, K), 0.5)
        weights = torch.randint(0, 5, (t, k), generator=g).float()
        out = run_down(hip, dev, "float", hh, experts, offsets, rows, w2, s2, weights, None)
        assert torch.equal(out, ref.down(hh, experts, offsets, rows, w2, s2, weights, None)[0].float())


def test_a_layer_from_router_to_sum(hip, dev):
    """Router, order, up, down, as a decoder's layer runs them; each against its statement on what the one before it gave.  Then captured and
    replayed with other inputs, on another stream, with eager work between."""
    t, e, k, H, I = 150, 16, 4, 256, 352
    name, dtype = "bfloat16", torch.bfloat16
    g = torch.Generator().manual_seed(1)
    w1 = (torch.randn(e, 2, I, H, generator=g) * 33).round().clamp(-127, 127).to(torch.int8)
    w2 = (torch.randn(e, 1, H, I, generator=g) * 33).round().clamp(-127, 127).to(torch.int8)
    s1, s2 = torch.rand(e, 2, I, generator=g) * 0.003, torch.rand(e, 1, H, generator=g) * 0.003
    p1, p2, s1d, s2d = pack(hip, dev, w1), pack(hip, dev, w2), s1.to(dev), s2.to(dev)
    router = torch.randn(H, e, generator=g) / 16
    rp = hip.route_params(hip.FLOAT, e, k, renormalise=True)
    ep = hip.experts_params(hip.BFLOAT16, e, k, t, H, I)
    x, logits = torch.empty(t, H, dtype=dtype, device=dev), torch.empty(t, e, device=dev)
    ids, w = torch.empty(t, k, dtype=torch.int32, device=dev), torch.empty(t, k, device=dev)
    offsets, rows = torch.empty(e + 1, dtype=torch.int32, device=dev), torch.empty(t * k, dtype=torch.int32, device=dev)
    h, out = torch.empty(t * k, I, dtype=dtype, device=dev), torch.empty(t, H, dtype=dtype, device=dev)
    ow = torch.empty(hip.group_rows_workspace(t * k, e), dtype=torch.uint8, device=dev)
    ew = torch.empty(hip.experts_workspace(ep), dtype=torch.uint8, device=dev)

    def step(stream):
        hip.route(rp, t, logits, None, ids, w, stream)
        hip.group_rows(t * k, e, ids, offsets, rows, ow, stream)
        hip.experts_up(ep, x, offsets, rows, p1, s1d, h, ew, stream)
        hip.experts_down(ep, h, ids, offsets, rows, p2, s2d, w, x, out, ew, stream)

    def load(seed):
        gg = torch.Generator().manual_seed(seed)
        xs = torch.randn(t, H, generator=gg).to(dtype)
        x.copy_(xs)
        logits.copy_(xs.float() @ router)

    load(10)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    step(side.cuda_stream)
    side.synchronize()
    want_ids, want_w = ref.route(logits.cpu(), None, k, "softmax", renormalise=True)
    assert torch.equal(ids.cpu(), want_ids)
    o, r = ref.order(want_ids, e)
    assert torch.equal(offsets.cpu(), o) and torch.equal(rows.cpu(), r)
    want_h = ref.up(x.cpu(), o, r, k, w1, s1, "swish", True)
    v = ref.up(x.cpu(), o, r, k, w1[:, 1:], s1[:, 1:], "none", False).abs() * (ref.up(x.cpu(), o, r, k, w1[:, :1], s1[:, :1], "none", False).abs() + 1)
    assert bool(((h.cpu().double() - want_h).abs() <= 2.0 ** -8 * want_h.abs() * (1 + 2.0 ** -10) + 40 * STEP * v).all())
    want, size = ref.down(h.cpu(), ids.cpu(), o, r, w2, s2, w.cpu(), x.cpu())
    assert bool(((out.cpu().double() - want).abs() <= 2.0 ** -8 * want.abs() * (1 + 2.0 ** -10) + (k + 6) * STEP * size).all())

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(torch.cuda.current_stream().cuda_stream)
    for seed in range(20, 24):
        load(seed)
        graph.replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in (ids, w, offsets, rows, h, out)]
        ew.fill_(0xff)
        step(0)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, (ids, w, offsets, rows, h, out)))


def test_a_workspace_for_more_tokens_serves_fewer(hip, dev):
    t, k, e, K, N = 300, 2, 4, 128, 96
    g = torch.Generator().manual_seed(2)
    w = whole((e, 1, N, K), 4, g).to(torch.int8)
    packed, scales = pack(hip, dev, w), torch.ones(e, 1, N, device=dev)
    large = hip.experts_workspace(hip.experts_params(hip.HALF, e, k, t, K, N))
    work = guarded(large, dev)
    for n in (t, 5, 64, 1):
        x = whole((n, K), 3, g, largest=127.0).half()
        experts = choices(n, k, e, n)
        offsets, rows = ref.order(experts, e)
        p = hip.experts_params(hip.HALF, e, k, n, K, N, activation=hip.ACT_NONE, gated=False)
        h = torch.empty(n * k, N, dtype=torch.float16, device=dev)
        hip.experts_up(p, x.to(dev), offsets.to(dev), rows.to(dev), packed, scales, h, work)
        torch.cuda.synchronize()
        assert torch.equal(h.cpu(), ref.up(x, offsets, rows, k, w, scales.cpu(), "none", False).half())
    assert bool((work[large:] == 0x5a).all())
