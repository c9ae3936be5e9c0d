"""A router's choice and the order of rows by group, against their statements in 64 bits.  Both sides rank in 64 bits: experts, offsets and
rows are compared exactly (inputs are such that no two ranks that differ lie within 1e-12 of one another, or they are equal), weights to half
a step of fp32 plus 64-bit arithmetic."""
import math

import pytest
import torch

from tests import chosen_reference as ref

pytestmark = pytest.mark.gpu


def type_of(hip, name):
    return {"float": hip.FLOAT, "bfloat16": hip.BFLOAT16, "half": hip.HALF}[name]


def route(hip, dev, logits, bias, k, score="softmax", stride=None, **kw):
    name = {torch.float32: "float", torch.bfloat16: "bfloat16", torch.float16: "half"}[logits.dtype]
    t, e = logits.shape
    p = hip.route_params(type_of(hip, name), e, k, score=hip.ROUTE_SIGMOID if score == "sigmoid" else hip.ROUTE_SOFTMAX, logits_stride=stride, **kw)
    ids, w = torch.full((t + 1, k), -7, dtype=torch.int32, device=dev), torch.full((t + 1, k), -7.0, device=dev)
    if stride is None:
        x = logits.to(dev)
    else:
        x = torch.full((t, stride), 99.0, dtype=logits.dtype, device=dev)
        x[:, :e] = logits.to(dev)
    hip.route(p, t, x, None if bias is None else bias.to(dev), ids, w)
    torch.cuda.synchronize()
    assert bool((ids[t] == -7).all()) and bool((w[t] == -7).all())
    return ids[:t].cpu(), w[:t].cpu()


def check(got, want):
    assert torch.equal(got[0], want[0]), (got[0] != want[0]).nonzero()[:4]
    w = want[1]
    assert torch.equal(got[1].isnan(), w.isnan())
    off = (got[1].double() - w).abs() - (2.0 ** -24 * w.abs() * (1 + 2.0 ** -20) + 2.0 ** -150)
    assert bool((off[~w.isnan()] <= 0).all()), float(off[~w.isnan()].max())


def logits_of(t, e, dtype, seed, spread=1.5):
    return (torch.randn(t, e, generator=torch.Generator().manual_seed(seed)) * spread).to(dtype)


@pytest.mark.parametrize("name", list(ref.TYPES))
@pytest.mark.parametrize("t,e,k", [(1, 1, 1), (1, 8, 2), (3, 4, 4), (17, 60, 4), (33, 64, 6), (5, 65, 8), (65, 128, 8), (7, 255, 32), (130, 256, 8), (9, 257, 3), (6, 1000, 32), (5, 1024, 8), (1030, 100, 8), (1500, 256, 5)])
@pytest.mark.parametrize("score,biased,renormalise", [("softmax", False, True), ("sigmoid", True, True), ("softmax", True, False)])
def test_route(hip, dev, name, t, e, k, score, biased, renormalise):
    x = logits_of(t, e, ref.TYPES[name], t * 1000 + e)
    bias = logits_of(1, e, torch.float32, 5, 0.1)[0] if biased else None
    kw = dict(renormalise=renormalise, scale=2.5 if renormalise else 1.0)
    check(route(hip, dev, x, bias, k, score, **kw), ref.route(x, bias, k, score, **kw))


@pytest.mark.parametrize("e,groups,top_groups,best,k", [(64, 8, 3, 2, 6), (256, 8, 4, 2, 8), (160, 8, 3, 1, 6), (60, 4, 2, 2, 4), (12, 3, 1, 1, 4), (64, 64, 8, 1, 8), (1024, 32, 4, 2, 32),
                                                       (510, 51, 7, 2, 9), (16, 1, 1, 1, 3), (63, 63, 63, 1, 32)])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_groups(hip, dev, e, groups, top_groups, best, k, score):
    for t in (37, 1100):
        groups_of_tokens(hip, dev, t, e, groups, top_groups, best, k, score)


def groups_of_tokens(hip, dev, t, e, groups, top_groups, best, k, score):
    x = logits_of(t, e, torch.float32, e + groups + t)
    bias = logits_of(1, e, torch.float32, 6, 0.3)[0]
    kw = dict(groups=groups, top_groups=top_groups, group_best=best, renormalise=True)
    check(route(hip, dev, x, bias, k, score, **kw), ref.route(x, bias, k, score, **kw))


@pytest.mark.parametrize("e", [8, 100, 256, 600])
def test_equal_scores_and_strides(hip, dev, e):
    """Many equal ranks: the lowest index first.  Whole numbers as logits; rows that lie apart, with large values between them."""
    x = torch.randint(-2, 3, (41, e), generator=torch.Generator().manual_seed(e)).to(torch.bfloat16)
    for score in ("softmax", "sigmoid"):
        check(route(hip, dev, x, None, 8, score, stride=e + 3), ref.route(x, None, 8, score))
    kw = dict(groups=4, top_groups=2, group_best=2)
    check(route(hip, dev, x, None, 4, "sigmoid", stride=e + 8, **kw), ref.route(x, None, 4, "sigmoid", **kw))
    zero = torch.zeros(3, e)
    got = route(hip, dev, zero, None, 5)
    assert torch.equal(got[0], torch.arange(5, dtype=torch.int32).expand(3, 5))


def test_what_is_not_finite(hip, dev):
    x = logits_of(12, 70, torch.float32, 1)
    inf, nan = math.inf, math.nan
    x[0, 3] = nan
    x[1, 3] = inf
    x[2, 3] = -inf
    x[3] = -inf
    x[4] = nan
    x[5, 4:] = -inf          # four experts are left for eight choices
    x[6] = 1e30
    x[7] = -1e30
    x[8, 0], x[8, 1] = 800.0, 30.0
    x[9, 20:] = 40.0         # sigmoid 1 - 4e-18: all the same in 64 bits
    x[10, 5:] = -800.0
    for score, renormalise in (("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)):
        check(route(hip, dev, x, None, 8, score, renormalise=renormalise), ref.route(x, None, 8, score, renormalise=renormalise))
    bias = torch.zeros(70)
    bias[7], bias[9], bias[11] = -inf, nan, inf
    for kw in (dict(), dict(groups=7, top_groups=3, group_best=2)):
        check(route(hip, dev, x, bias, 8, "sigmoid", **kw), ref.route(x, bias, 8, "sigmoid", **kw))


def order(hip, dev, group_of, groups):
    n = group_of.numel()
    offsets, rows = torch.full((groups + 2,), -7, dtype=torch.int32, device=dev), torch.full((n + 1,), -7, dtype=torch.int32, device=dev)
    size = hip.group_rows_workspace(n, groups)
    work = torch.full((size + 16,), 0x5a, dtype=torch.uint8, device=dev)
    hip.group_rows(n, groups, group_of.to(dev), offsets, rows, work)
    torch.cuda.synchronize()
    assert int(offsets[-1]) == -7 and int(rows[-1]) == -7 and bool((work[size:] == 0x5a).all())
    return offsets[:-1].cpu(), rows[:-1].cpu()


@pytest.mark.parametrize("n", [0, 1, 2, 63, 64, 65, 255, 256, 257, 1000, 1023, 1024, 1025, 2048, 3000, 8192, 65536, 70001, 300000])
@pytest.mark.parametrize("groups", [1, 2, 8, 60, 256, 1023, 1024])
def test_group_rows(hip, dev, n, groups):
    g = torch.Generator().manual_seed(n + groups)
    of = torch.randint(-2, groups + 2, (n,), generator=g, dtype=torch.int32)
    offsets, rows = order(hip, dev, of, groups)
    key = torch.where((of < 0) | (of >= groups), groups, of).long()
    assert torch.equal(rows.long(), torch.sort(key, stable=True)[1])
    counts = torch.bincount(key, minlength=groups + 1)[:groups]
    assert torch.equal(offsets.long(), torch.cat([torch.zeros(1, dtype=torch.long), counts.cumsum(0)]))


def test_group_rows_of_one_group_and_of_none(hip, dev):
    for n in (5, 5000):
        for value, where in ((0, n), (3, 0), (-1, 0), (2 ** 31 - 1, 0), (-2 ** 31, 0)):
            of = torch.full((n,), value, dtype=torch.int32)
            offsets, rows = order(hip, dev, of, 2)
            assert torch.equal(rows, torch.arange(n, dtype=torch.int32)) and offsets.tolist() == [0, where, where]
    assert order(hip, dev, torch.tensor([3, 0, 1, 0, 9, 1], dtype=torch.int32), 3)[0].tolist() == ref.order(torch.tensor([3, 0, 1, 0, 9, 1]), 3)[0].tolist()


def test_a_captured_choice_follows_its_inputs(hip, dev):
    """Router and order in a graph, on another stream, replayed with other logits and with eager work between."""
    t, e, k = 700, 64, 6
    p = hip.route_params(hip.FLOAT, e, k, renormalise=True)
    x = torch.zeros(t, e, device=dev)
    ids, w = torch.empty(t, k, dtype=torch.int32, device=dev), torch.empty(t, k, device=dev)
    offsets, rows = torch.empty(e + 1, dtype=torch.int32, device=dev), torch.empty(t * k, dtype=torch.int32, device=dev)
    work = torch.empty(hip.group_rows_workspace(t * k, e), dtype=torch.uint8, device=dev)

    def step(stream):
        hip.route(p, t, x, None, ids, w, stream)
        hip.group_rows(t * k, e, ids, offsets, rows, work, stream)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(side.cuda_stream)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(torch.cuda.current_stream().cuda_stream)
    for seed in range(4):
        logits = logits_of(t, e, torch.float32, 50 + seed)
        x.copy_(logits)
        graph.replay()
        torch.cuda.synchronize()
        got = [v.clone() for v in (ids, w, offsets, rows)]
        want = ref.route(logits, None, k, "softmax", renormalise=True)
        check((got[0].cpu(), got[1].cpu()), want)
        step(0)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, (ids, w, offsets, rows)))
        key = got[0].reshape(-1).cpu().long()
        assert torch.equal(got[3].cpu().long(), torch.sort(key, stable=True)[1])
