"""Low-rank adapters, against their statement in 64 bits.

Whole numbers are exact: x A^T stays below 2^16, which two bfloat16 numbers hold, sums below 2^24, so that a result is one rounding of a whole number.
Elsewhere: a sum of K products over chains of K / 32 matrix instructions, each a few roundings, and of shares: (K / 32 + 48) 2^-24 of what its terms
add up to in absolute value; x A^T as two numbers of the type, 2^-16 of it in bfloat16, 2^-22 of the row's largest in half precision (covered by
2^-20 of the terms' sum where ranks are 8 and more and rows' values alike); the last sum and its scaling 6 steps; the type's rounding, eps / 2."""
import math

import pytest
import torch

from tests import chosen_reference as ref

pytestmark = pytest.mark.gpu
STEP = 2.0 ** -24


def type_of(hip, name):
    return {"float": hip.FLOAT, "bfloat16": hip.BFLOAT16, "half": hip.HALF}[name]


def run(hip, dev, name, x, offsets, rows, a, b, ranks, scales, base, ends, rank, in_place=False, gaps=(0, 0, 0), stream=0, lead=0):
    t, k = x.shape
    n = ends[-1]
    p = hip.adapters_params(type_of(hip, name), a.shape[0], rank, t, k, ends, x_stride=k + gaps[0], base_stride=n + gaps[1],
                            out_stride=n + (gaps[1] if in_place else gaps[2]))

    def placed(v, gap):
        flat = torch.full((lead + v.shape[0] * (v.shape[1] + gap),), 11.0, dtype=v.dtype, device=dev)
        flat[lead:].view(v.shape[0], -1)[:, :v.shape[1]] = v.to(dev)
        return flat

    xd, bd = placed(x, gaps[0]), placed(base, gaps[1])
    out = bd if in_place else placed(torch.full_like(base, 7.0), gaps[2])
    size = hip.adapters_workspace(p)
    work = torch.full((size + 64,), 0x5a, dtype=torch.uint8, device=dev)
    up = lambda v: None if v is None else v.to(dev)
    hip.adapters(p, xd[lead:], offsets.to(dev), rows.to(dev), a.to(dev), b.to(dev), up(ranks), scales.to(dev), bd[lead:], out[lead:], work, stream)
    torch.cuda.synchronize()
    assert bool((work[size:] == 0x5a).all())
    got = out[lead:].view(t, -1)
    assert bool((got[:, n:] == 11).all()) and bool((out[:lead] == 11).all())
    return got[:, :n].cpu()


def whole(shape, limit, g):
    return torch.randint(-limit, limit + 1, shape, generator=g).float()


SIZES = [  # tokens, adapters, rank, K, ends, ragged ranks
    (1, 1, 8, 8, [1], False), (1, 4, 16, 64, [64], False), (2, 2, 8, 40, [100], False), (7, 3, 24, 72, [64, 96, 131], True), (16, 1, 32, 256, [130], False),
    (17, 5, 64, 200, [33, 34, 97, 200], True), (64, 64, 16, 512, [256, 320, 384], True), (65, 2, 40, 1040, [70], False), (100, 1000, 8, 64, [48], False),
    (300, 3, 128, 96, [300], True), (33, 2, 256, 64, [128], True), (1000, 5, 16, 160, [513], False), (5, 3, 16, 4104, [64], False), (2100, 4, 64, 320, [200], False),
    (4500, 2, 16, 96, [4100], False), (4500, 2, 24, 96, [4100], True), (40, 3, 16, 2048, [1030, 2100], True), (20, 20, 8, 2056, [1024], False), (4200, 3, 72, 72, [1030, 2070], True), (4200, 1, 256, 64, [2100], False)]


@pytest.mark.parametrize("name", list(ref.TYPES))
@pytest.mark.parametrize("t,n,rank,K,ends,ragged", SIZES)
def test_exactly(hip, dev, name, t, n, rank, K, ends, ragged):
    g = torch.Generator().manual_seed(t + K)
    dtype = ref.TYPES[name]
    x, a, b = whole((t, K), 2, g).to(dtype), whole((n, len(ends) * rank, K), 2, g).to(dtype), whole((n, ends[-1], rank), 3, g).to(dtype)
    base, scales = whole((t, ends[-1]), 64, g).to(dtype), torch.randint(1, 4, (n,), generator=g).float()
    ranks = torch.randint(0, rank + 5, (n,), generator=g, dtype=torch.int32) if ragged else None
    of = torch.randint(-1, n, (t,), generator=g)
    if t > 64:
        of = of.sort()[0]
    offsets, rows = ref.order(of, n)
    if name == "half":     # the row's largest has 22 bits, which covers all of them
        assert K * 4 < 2 ** 20
    want, size = ref.adapters(x, offsets, rows, a, b, ranks, scales, base, ends, rank)
    assert float(want.abs().max()) < 2 ** 24 and K * 4 < 2 ** 16
    fits = want.abs() < torch.finfo(dtype).max
    got = run(hip, dev, name, x, offsets, rows, a, b, ranks, scales, base, ends, rank)
    assert torch.equal(got[fits], want.float().to(dtype)[fits]), (got.double() - want)[fits].abs().max()
    # in place, rows apart, at odd addresses: the same bits
    again = run(hip, dev, name, x, offsets, rows, a, b, ranks, scales, base, ends, rank, in_place=True, gaps=(3, 5, 0), lead=1)
    assert torch.equal(again, got)
    again = run(hip, dev, name, x, offsets, rows, a, b, ranks, scales, base, ends, rank, gaps=(8, 16, 24), lead=8)
    assert torch.equal(again, got)


@pytest.mark.parametrize("name", list(ref.TYPES))
@pytest.mark.parametrize("K", [50, 77, 1003])
def test_odd_widths_of_x(hip, dev, name, K):
    g = torch.Generator().manual_seed(K)
    dtype, rank, ends, t, n = ref.TYPES[name], 16, [30, 61], 20, 3
    x, a, b = whole((t, K), 2, g).to(dtype), whole((n, 2 * rank, K), 2, g).to(dtype), whole((n, 61, rank), 3, g).to(dtype)
    base, scales = whole((t, 61), 64, g).to(dtype), torch.ones(n)
    offsets, rows = ref.order(torch.randint(0, n, (t,), generator=g), n)
    want, _ = ref.adapters(x, offsets, rows, a, b, None, scales, base, ends, rank)
    assert torch.equal(run(hip, dev, name, x, offsets, rows, a, b, None, scales, base, ends, rank), want.float().to(dtype))


@pytest.mark.parametrize("name", list(ref.TYPES))
@pytest.mark.parametrize("t,n,rank,K,ends", [(1, 2, 16, 4096, [512]), (40, 40, 16, 2048, [256, 320]), (500, 3, 64, 1024, [300])])
def test_against_64_bits(hip, dev, name, t, n, rank, K, ends):
    g = torch.Generator().manual_seed(t)
    dtype = ref.TYPES[name]
    x = torch.randn(t, K, generator=g).to(dtype)
    a, b = (torch.randn(n, len(ends) * rank, K, generator=g) * K ** -0.5).to(dtype), (torch.randn(n, ends[-1], rank, generator=g) * 0.1).to(dtype)
    base, scales = torch.randn(t, ends[-1], generator=g).to(dtype), torch.rand(n, generator=g) + 0.5
    offsets, rows = ref.order(torch.randint(-1, n, (t,), generator=g), n)
    got = run(hip, dev, name, x, offsets, rows, a, b, None, scales, base, ends, rank).double()
    want, size = ref.adapters(x, offsets, rows, a, b, None, scales, base, ends, rank)
    held = {"float": 0.0, "bfloat16": 2.0 ** -16, "half": 2.0 ** -20}[name]
    tol = ((K / 32 + 48 + 6) * STEP + held) * size + torch.finfo(dtype).eps / 2 * want.abs() * (1 + 2.0 ** -10) + torch.finfo(dtype).tiny * 2.0 ** -10
    off = (got - want).abs() - tol
    assert bool((off <= 0).all()), float(off.max())


def test_values_of_any_size_in_half_precision(hip, dev):
    """x A^T beyond a half's range, and far below it."""
    t, rank, K, N = 6, 16, 256, 64
    g = torch.Generator().manual_seed(0)
    x, a = torch.randn(t, K, generator=g).half(), torch.randn(1, rank, K, generator=g).half()
    x[1] *= 1000
    x[2] = (x[2].float() * 1e-4).half()
    x[3] = 0
    b = torch.randn(1, N, rank, generator=g).half()
    a *= 16
    base, scales = torch.zeros(t, N).half(), torch.tensor([2.0 ** -10])
    offsets, rows = torch.tensor([0, t], dtype=torch.int32), torch.arange(t, dtype=torch.int32)
    got = run(hip, dev, "half", x, offsets, rows, a, b, None, scales, base, [N], rank).double()
    want, size = ref.adapters(x, offsets, rows, a, b, None, scales, base, [N], rank)
    tol = ((K / 32 + 54) * STEP + 2.0 ** -20) * size + 2.0 ** -11 * want.abs() * (1 + 2.0 ** -10) + 2.0 ** -25
    assert float((x[1].double() @ a[0].double().T).abs().max()) > 65504 and bool(((got - want).abs() <= tol).all())


def test_what_is_not_read_and_what_is_not_finite(hip, dev):
    """NaN beyond an adapter's rank, in other adapters and in other tokens stays where it is."""
    t, n, rank, K, ends = 9, 3, 16, 64, [40, 90]
    g = torch.Generator().manual_seed(4)
    for name, dtype in ref.TYPES.items():
        x, a, b = whole((t, K), 2, g).to(dtype), whole((n, 2 * rank, K), 2, g).to(dtype), whole((n, 90, rank), 2, g).to(dtype)
        base, scales, ranks = whole((t, 90), 9, g).to(dtype), torch.ones(n), torch.tensor([16, 5, 0], dtype=torch.int32)
        offsets, rows = ref.order(torch.tensor([0, 1, 2, -1, 0, 1, 2, 7, 1]), n)
        want, _ = ref.adapters(x, offsets, rows, a, b, ranks, scales, base, ends, rank)
        for g2, r in ((1, 5), (2, 0)):
            a.view(n, 2, rank, K)[g2, :, r:] = math.nan
            b[g2, :, r:] = math.nan
        scales[2] = 1.0
        got = run(hip, dev, name, x, offsets, rows, a, b, ranks, scales, base, ends, rank)
        assert torch.equal(got, want.float().to(dtype)), name
        x[0, 3], x[3, 1] = math.nan, math.inf          # a token of adapter 0; one without an adapter
        got = run(hip, dev, name, x, offsets, rows, a, b, ranks, scales, base, ends, rank)
        assert bool((~got[0].isfinite()).all()) and torch.equal(got[1:], want[1:].float().to(dtype)), name


@pytest.mark.parametrize("rank,K", [(16, 64), (8, 40), (16, 4096), (32, 64)])
def test_an_adapter_of_no_rank_adds_nothing(hip, dev, rank, K):
    """whatever its tokens hold: x A^T has no columns then"""
    t, ends = 5, [40, 90]
    g = torch.Generator().manual_seed(6)
    for name, dtype in ref.TYPES.items():
        x, a, b = whole((t, K), 2, g).to(dtype), whole((2, 2 * rank, K), 2, g).to(dtype), whole((2, 90, rank), 2, g).to(dtype)
        x[0, 3], x[2, 1] = math.nan, math.inf
        base, ranks = whole((t, 90), 9, g).to(dtype), torch.tensor([0, 3], dtype=torch.int32)
        offsets, rows = ref.order(torch.tensor([0, 1, 0, 1, 0]), 2)
        got = run(hip, dev, name, x, offsets, rows, a, b, ranks, torch.ones(2), base, ends, rank)
        assert torch.equal(got[[0, 2, 4]], base[[0, 2, 4]]), name


def test_beside_a_quantized_linear_and_captured(hip, dev):
    """A quantized linear's output gets its adapters in place, eagerly on another stream and in a graph that is replayed with other tokens."""
    t, n, rank, K, N = 20, 4, 16, 256, 192
    g = torch.Generator().manual_seed(9)
    w = whole((K, N), 100, g).to(torch.int8).to(dev)
    packed, sums = torch.empty(hip.qgemm_packed_bytes(K, N), dtype=torch.int8, device=dev), torch.empty(N, dtype=torch.int32, device=dev)
    hip.qgemm_prepack_b(w, False, K, N, packed, sums)
    mx = torch.full((1,), 0.5, device=dev)
    mn, zero = -mx, torch.zeros(N, device=dev)
    a, b = (torch.randn(n, rank, K, generator=g) / 16).to(dev), torch.randn(n, N, rank, generator=g).to(dev)
    scales = torch.ones(n, device=dev)
    x, xq = torch.empty(t, K, device=dev), torch.empty(t, K, dtype=torch.uint8, device=dev)
    state, out = torch.empty(hip.DYNAMIC_STATE_FLOATS, device=dev), torch.empty(t, N, device=dev)
    of, offsets, rows = (torch.empty(s, dtype=torch.int32, device=dev) for s in (t, n + 1, t))
    p = hip.adapters_params(hip.FLOAT, n, rank, t, K, [N])
    work = torch.empty(hip.adapters_workspace(p), dtype=torch.uint8, device=dev)
    ow = torch.empty(hip.group_rows_workspace(t, n), dtype=torch.uint8, device=dev)
    mp = hip.matmul_params(api=hip.API_V2, t_in=hip.QUINT8, t_out=hip.FLOAT, input_mode=hip.MIN_FIRST, has_dequantize=True)

    def linear(stream):
        hip.quantize_dynamic(x, xq, t * K, hip.QUINT8, hip.MIN_FIRST, 0.01, state, stream)
        hip.qmatmul_device_range(mp, xq, packed, sums, t, K, N, state.data_ptr() + 8, mn, mx, 1, zero, out, stream)

    def step(stream):
        linear(stream)
        hip.group_rows(t, n, of, offsets, rows, ow, stream)
        hip.adapters(p, x, offsets, rows, a, b, None, scales, out, out, work, stream)

    def load(seed):
        gg = torch.Generator().manual_seed(seed)
        x.copy_(torch.randn(t, K, generator=gg))
        of.copy_(torch.randint(-1, n, (t,), generator=gg, dtype=torch.int32))
        torch.cuda.synchronize()

    load(1)
    linear(0)
    torch.cuda.synchronize()
    base = out.cpu().clone()
    side = torch.cuda.Stream()
    step(side.cuda_stream)
    side.synchronize()
    want, size = ref.adapters(x.cpu(), offsets.cpu(), rows.cpu(), a.cpu(), b.cpu(), None, scales.cpu(), base, [N], rank)
    assert bool(((out.cpu().double() - want).abs() <= (K / 32 + 54) * STEP * size + STEP * want.abs()).all())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(torch.cuda.current_stream().cuda_stream)
    for seed in range(5, 9):
        load(seed)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        step(0)
        torch.cuda.synchronize()
        assert torch.equal(got, out)


def test_orders_that_are_none_stay_inside(hip, dev):
    t, n, rank, K, N = 9, 3, 8, 64, 64
    p = hip.adapters_params(hip.FLOAT, n, rank, t, K, [N])
    for offsets in ([0, 5, 100, 9], [-4, 7, 3, 1 << 30], [9, 9, 9, 9], [0, 9, 0, 9], [9, 0, 9, 0]):
        rows = torch.tensor([0, 8, 9, -1, 1 << 30, 3, 3, 3, 3], dtype=torch.int32, device=dev)
        out, size = torch.zeros(t + 1, N, device=dev), hip.adapters_workspace(p)
        work = torch.full((size + 64,), 0x5a, dtype=torch.uint8, device=dev)
        hip.adapters(p, torch.ones(t, K, device=dev), torch.tensor(offsets, dtype=torch.int32, device=dev), rows, torch.ones(n, rank, K, device=dev),
                     torch.ones(n, N, rank, device=dev), torch.tensor([8, 1 << 30, -5], dtype=torch.int32, device=dev), torch.ones(n, device=dev),
                     torch.zeros(t, N, device=dev), out, work)
        torch.cuda.synchronize()
        assert bool((out[-1] == 0).all()) and bool((work[size:] == 0x5a).all())
