"""Adapters of many tokens whose x A^T is made in several shares of K: tiles of 64 places, each share in a part of the workspace of its own, the product with B
adding them up while the next rows are on their way.

Tolerances are those of test_gpu_adapters.py: whole numbers are exact; elsewhere (K / 32 + 48 + 6) 2^-24 of what the terms add up to in absolute value,
x A^T as two numbers of the type, and the result's rounding, eps / 2."""
import pytest
import torch

from tests import chosen_reference as ref
from tests.test_gpu_adapters import STEP, run, whole

pytestmark = pytest.mark.gpu

SIZES = [  # tokens, adapters, rank, K, ends, ragged ranks
    (4500, 2, 64, 1024, [4100], False), (4300, 3, 32, 1096, [1030, 2070, 4200], True), (4200, 5, 16, 776, [4120], False), (5000, 2, 24, 2304, [700, 2104], True),
    (9000, 9, 128, 520, [4200], True), (4500, 4, 16, 776, [300], False)]


def inputs(t, n, rank, ends, ragged, g):
    ranks = torch.randint(0, rank + 5, (n,), generator=g, dtype=torch.int32) if ragged else None
    of = torch.randint(-1, n, (t,), generator=g).sort()[0]
    return ranks, ref.order(of[torch.randperm(t, generator=g)], n)


@pytest.mark.parametrize("name", list(ref.TYPES))
@pytest.mark.parametrize("t,n,rank,K,ends,ragged", SIZES)
def test_exactly(hip, dev, name, t, n, rank, K, ends, ragged):
    g = torch.Generator().manual_seed(t + K)
    dtype = ref.TYPES[name]
    x, a, b = whole((t, K), 2, g).to(dtype), whole((n, len(ends) * rank, K), 2, g).to(dtype), whole((n, ends[-1], rank), 3, g).to(dtype)
    base, scales = whole((t, ends[-1]), 64, g).to(dtype), torch.randint(1, 4, (n,), generator=g).float()
    ranks, (offsets, rows) = inputs(t, n, rank, ends, ragged, g)
    want, _ = ref.adapters(x, offsets, rows, a, b, ranks, scales, base, ends, rank)
    assert float(want.abs().max()) < 2 ** 24 and K * 4 < 2 ** 16
    fits = want.abs() < torch.finfo(dtype).max
    got = run(hip, dev, name, x, offsets, rows, a, b, ranks, scales, base, ends, rank)
    assert torch.equal(got[fits], want.float().to(dtype)[fits]), (got.double() - want)[fits].abs().max()
    again = run(hip, dev, name, x, offsets, rows, a, b, ranks, scales, base, ends, rank, in_place=True, gaps=(3, 5, 0), lead=1)
    assert torch.equal(again, got)


@pytest.mark.parametrize("name", list(ref.TYPES))
@pytest.mark.parametrize("t,n,rank,K,ends", [(4500, 2, 64, 1024, [2100]), (4300, 3, 32, 1096, [1030, 2070])])
def test_against_64_bits(hip, dev, name, t, n, rank, K, ends):
    g = torch.Generator().manual_seed(t)
    dtype = ref.TYPES[name]
    x = torch.randn(t, K, generator=g).to(dtype)
    a, b = (torch.randn(n, len(ends) * rank, K, generator=g) * K ** -0.5).to(dtype), (torch.randn(n, ends[-1], rank, generator=g) * 0.1).to(dtype)
    base, scales = torch.randn(t, ends[-1], generator=g).to(dtype), torch.rand(n, generator=g) + 0.5
    _, (offsets, rows) = inputs(t, n, rank, ends, False, g)
    got = run(hip, dev, name, x, offsets, rows, a, b, None, scales, base, ends, rank).double()
    want, size = ref.adapters(x, offsets, rows, a, b, None, scales, base, ends, rank)
    held = {"float": 0.0, "bfloat16": 2.0 ** -16, "half": 2.0 ** -20}[name]
    tol = ((K / 32 + 48 + 6) * STEP + held) * size + torch.finfo(dtype).eps / 2 * want.abs() * (1 + 2.0 ** -10) + torch.finfo(dtype).tiny * 2.0 ** -10
    off = (got - want).abs() - tol
    assert bool((off <= 0).all()), float(off.max())
