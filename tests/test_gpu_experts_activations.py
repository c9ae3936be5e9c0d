"""The activations of the experts' products through every kernel that has them, gated and not, with rows that are not finite among the others;
and the way back with such rows through tiles.

Tolerances are those of test_gpu_experts.py: a value v = fp32(sum) * (s * scale) has three roundings, 3 2^-24 |v|; an activation y of it follows with its
slope (at most 1.13) and its own evaluation, (16 + 8 |a|) 2^-24 |y| for swish and the tanh gelu (a: the argument of their exponential), 1e-6 + 2e-6 |y| for the erf
gelu; the product with v1 adds 4 steps; the result is rounded to its type, eps / 2."""
import math

import pytest
import torch

from tests import chosen_reference as ref
from tests.test_gpu_experts import STEP, choices, run_down, run_up

pytestmark = pytest.mark.gpu

# kernel: tokens, top_k, experts, K, N
SIZES = {
    "fused strips of 8": (6, 2, 5, 530, 150),
    "fused strips of 4": (16, 2, 64, 64, 1100),
    "strips": (40, 2, 5, 530, 150),
    "tiles of 128": (900, 2, 5, 530, 1100),
    "tiles of 128, long rows": (400, 2, 4, 2000, 1100),
    "tiles of 256": (3200, 2, 16, 200, 2100),
}
CASES = [(kernel, activation, name) for kernel in SIZES for activation in ("swish", "gelu_approx", "gelu_exact", "relu", "none") for name in ref.TYPES
         if kernel != "tiles of 256" or (activation in ("swish", "relu") and name != "half")]   # (the one that has a kernel of its own there, and one that has none)


def spoiled(x, g):
    """Some rows with a NaN or an infinity, at the first and the last element too"""
    n = len(x)
    for i, value in enumerate((math.nan, math.inf, -math.inf, math.nan)):
        at = (0, x.shape[1] - 1, x.shape[1] // 2, 1)[i]
        x[(n - 1, n // 2, 0, n // 3)[i], at] = value
    return x


@pytest.mark.parametrize("gated", [True, False])
@pytest.mark.parametrize("kernel,activation,name", CASES)
def test_up(hip, dev, kernel, activation, name, gated):
    t, k, e, K, N = SIZES[kernel]
    g = torch.Generator().manual_seed(t + K)
    x = spoiled(torch.randn(t, K, generator=g) * (torch.randn(1, K, generator=g) * 0.5).exp(), g).to(ref.TYPES[name])
    w = (torch.randn(e, 1 + gated, N, K, generator=g) * 33).round().clamp(-127, 127).to(torch.int8)
    scales = (0.8 + 0.4 * torch.rand(e, 1 + gated, N, generator=g)) * (0.05 / K ** 0.5)
    offsets, rows = ref.order(choices(t, k, e, t), e)
    got = run_up(hip, dev, name, x, offsets, rows, k, w, scales, activation, gated).double()
    v0 = ref.up(x, offsets, rows, k, w[:, :1], scales[:, :1], "none", False)
    v1 = ref.up(x, offsets, rows, k, w[:, 1:], scales[:, 1:], "none", False) if gated else torch.ones_like(v0)
    y = ref.activate(activation, v0)
    a = {"swish": v0.abs(), "gelu_approx": 1.6 * v0.abs() * (1 + 0.045 * v0 ** 2)}.get(activation, torch.zeros_like(v0))
    own = 1e-6 + 2e-6 * y.abs() if activation == "gelu_exact" else (16 + 8 * a) * STEP * y.abs() if activation in ("swish", "gelu_approx") else 0.0 * y
    dy = 1.13 * 3 * STEP * v0.abs() + own
    want = y * v1
    bad = ~torch.isfinite(x[rows.long() // k]).all(-1)
    assert int(bad.sum()) == 4 * k and bool(got[bad].isnan().all()) and bool(got[~bad].isfinite().all())
    tol = dy * v1.abs() + 4 * STEP * want.abs() + torch.finfo(ref.TYPES[name]).eps / 2 * want.abs() * (1 + 2.0 ** -10) + torch.finfo(ref.TYPES[name]).tiny * 2.0 ** -10
    off = ((got - want).abs() - tol)[~bad]
    assert bool((off <= 0).all()), float(off.max())


@pytest.mark.parametrize("name", list(ref.TYPES))
def test_down_through_tiles(hip, dev, name):
    """A row that is not finite reaches its own token only."""
    t, k, e, K, N = 1500, 2, 3, 256, 600
    g = torch.Generator().manual_seed(11)
    h = spoiled(torch.randn(t * k, K, generator=g) * torch.randn(t * k, 1, generator=g).exp(), g).to(ref.TYPES[name])
    w = (torch.randn(e, 1, N, K, generator=g) * 33).round().clamp(-127, 127).to(torch.int8)
    scales = (0.8 + 0.4 * torch.rand(e, 1, N, generator=g)) * (0.03 / K ** 0.5)
    weights = torch.softmax(torch.randn(t, k, generator=g), -1)
    experts = choices(t, k, e, 5)
    offsets, rows = ref.order(experts, e)
    addend = torch.randn(t, N, generator=g).to(ref.TYPES[name])
    got = run_down(hip, dev, name, h, experts, offsets, rows, w, scales, weights, addend).double()
    want, size = ref.down(h, experts, offsets, rows, w, scales, weights, addend)
    bad = torch.zeros(t, dtype=torch.bool)
    bad[rows[~torch.isfinite(h).all(-1)].long() // k] = True
    assert bool(got[bad].isnan().all()) and bool(got[~bad].isfinite().all())
    tol = (4 + k + 2) * STEP * size + torch.finfo(ref.TYPES[name]).eps / 2 * want.abs() * (1 + 2.0 ** -10) + torch.finfo(ref.TYPES[name]).tiny * 2.0 ** -10
    off = ((got - want).abs() - tol)[~bad]
    assert bool((off <= 0).all()), float(off.max())
