"""Choices as uneven as they can be: kernels are chosen by the average number of rows a group, and have to be right for any.  Whole numbers, compared exactly;
and buffers that are aligned to their elements only."""
import pytest
import torch

from tests import chosen_reference as ref
from tests import test_gpu_adapters as adapters
from tests.test_gpu_experts import act_of, pack, run_down, run_up, type_of, whole

pytestmark = pytest.mark.gpu

# what every token chooses: one expert only, the first and the last one, one token another one, none of this device, one token here
def chosen(what, t, k, e):
    if what == "one":
        ids = torch.full((t, k), e // 2)
    elif what == "ends":
        ids = torch.zeros(t, k, dtype=torch.long)
        ids[t // 3:] = e - 1
    elif what == "but one":
        ids = torch.full((t, k), e - 1)
        ids[t // 2, 0] = 0
    else:
        ids = torch.full((t, k), e + 3)
        if what == "one here":
            ids[t - 1, k - 1] = 1
    return ids.to(torch.int32)


@pytest.mark.parametrize("name", list(ref.TYPES))
@pytest.mark.parametrize("what", ["one", "ends", "but one", "none here", "one here"])
@pytest.mark.parametrize("t,k,e,K,N", [(5, 1, 4, 64, 40), (300, 2, 8, 128, 96), (1500, 2, 3, 256, 600), (1700, 1, 4, 320, 1100), (2, 2, 8, 1440, 70)])
def test_experts(hip, dev, name, what, t, k, e, K, N):
    g = torch.Generator().manual_seed(t + K)
    experts = chosen(what, t, k, e)
    offsets, rows = ref.order(experts, e)
    x = whole((t, K), 3, g, largest=127.0).to(ref.TYPES[name])
    w = whole((e, 2, N, K), 4, g).to(torch.int8)
    scales = torch.full((e, 2, N), 2.0 ** -6)
    here = int(offsets[-1])
    want = ref.up(x, offsets, rows, k, w, scales, "none", True)[:here]
    got = run_up(hip, dev, name, x, offsets, rows, k, w, scales, "none", True)[:here]
    assert torch.equal(got, want.float().to(got.dtype))
    h = whole((t * k, K), 3, g, largest=127.0).to(ref.TYPES[name])
    weights, addend = torch.randint(0, 5, (t, k), generator=g).float(), whole((t, N), 100, g).to(ref.TYPES[name])
    want, _ = ref.down(h, experts, offsets, rows, w[:, :1], scales[:, :1] * 16, weights, addend)
    got = run_down(hip, dev, name, h, experts, offsets, rows, w[:, :1].contiguous(), (scales[:, :1] * 16).contiguous(), weights, addend)
    assert torch.equal(got, want.float().to(got.dtype))


@pytest.mark.parametrize("name", list(ref.TYPES))
@pytest.mark.parametrize("what", ["one", "ends", "none here", "one here"])
@pytest.mark.parametrize("t,n,rank,K,ends", [(9, 4, 16, 64, [40]), (9, 4, 24, 64, [40, 90]), (4500, 4, 16, 520, [1030]), (4500, 3, 64, 520, [4100])])
def test_adapters(hip, dev, name, what, t, n, rank, K, ends):
    g = torch.Generator().manual_seed(t + K)
    dtype = ref.TYPES[name]
    offsets, rows = ref.order(chosen(what, t, 1, n), n)
    x, a, b = whole((t, K), 2, g).to(dtype), whole((n, len(ends) * rank, K), 2, g).to(dtype), whole((n, ends[-1], rank), 3, g).to(dtype)
    base, scales = whole((t, ends[-1]), 64, g).to(dtype), torch.randint(1, 4, (n,), generator=g).float()
    want, _ = ref.adapters(x, offsets, rows, a, b, None, scales, base, ends, rank)
    fits = want.abs() < torch.finfo(dtype).max
    for in_place in (False, True):
        got = adapters.run(hip, dev, name, x, offsets, rows, a, b, None, scales, base, ends, rank, in_place=in_place)
        assert torch.equal(got[fits], want.float().to(dtype)[fits])


@pytest.mark.parametrize("name", list(ref.TYPES))
@pytest.mark.parametrize("t,k,e,K,N", [(5, 1, 4, 64, 64), (300, 2, 8, 128, 96), (1500, 2, 3, 256, 600)])
def test_experts_at_addresses_of_elements(hip, dev, name, t, k, e, K, N):
    """x, h, addend and out one element behind a 16-byte address, everything else one word behind it."""
    g = torch.Generator().manual_seed(t)
    dtype = ref.TYPES[name]
    experts = torch.randint(0, e + 2, (t, k), generator=g, dtype=torch.int32)
    offsets, rows = ref.order(experts, e)
    here = int(offsets[-1])

    def off(v):
        flat = torch.empty(v.numel() + 1, dtype=v.dtype, device=dev)
        flat[1:] = v.reshape(-1).to(dev)
        return flat[1:].view(v.shape)

    x, w = whole((t, K), 3, g, largest=127.0).to(dtype), whole((e, 1, N, K), 4, g).to(torch.int8)
    scales = torch.full((e, 1, N), 0.25)
    p = hip.experts_params(type_of(hip, name), e, k, t, K, N, activation=act_of(hip, "none"), gated=False)
    work = torch.empty(hip.experts_workspace(p), dtype=torch.uint8, device=dev)
    h = off(torch.full((t * k + 1, N), 7.0, dtype=dtype))
    hip.experts_up(p, off(x), off(offsets), off(rows), pack(hip, dev, w), off(scales), h, work)
    torch.cuda.synchronize()
    assert torch.equal(h[:here].cpu(), ref.up(x, offsets, rows, k, w, scales, "none", False)[:here].float().to(dtype)) and bool((h[here:] == 7).all())
    back = whole((t * k, N), 3, g, largest=127.0).to(dtype)
    w2, s2 = whole((e, 1, K, N), 4, g).to(torch.int8), torch.full((e, 1, K), 0.25)
    weights, addend = torch.randint(0, 5, (t, k), generator=g).float(), whole((t, K), 100, g).to(dtype)
    out = off(torch.full((t + 1, K), 7.0, dtype=dtype))
    hip.experts_down(p, off(back), off(experts), off(offsets), off(rows), pack(hip, dev, w2), off(s2), off(weights), off(addend), out, work)
    torch.cuda.synchronize()
    want, _ = ref.down(back, experts, offsets, rows, w2, s2, weights, addend)
    assert torch.equal(out[:t].cpu(), want.float().to(dtype)) and bool((out[t] == 7).all())
