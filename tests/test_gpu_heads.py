"""Norm and rotation of heads, appending to the 4-bit cache and reading it back, against their statements in 64 bits.

Tolerance of a float result r whose head holds values up to m: half a step of the type, eps / 2 |r|, plus fp32 arithmetic before it: a
norm's sum of up to 256 squares in partial sums of at most 16 (16 + 5 roundings, half of them in the root), three roundings of
the scaling, cosine and sine to 2e-7, three roundings of the rotation: under 24 steps of 2^-24 m times the attention factor.
Codes and parameters go through 64 bits on both sides: what the cache holds is compared exactly."""
import math

import pytest
import torch

from tests import kv4_reference as ref

pytestmark = pytest.mark.gpu
TYPES = {"float": torch.float32, "bfloat16": torch.bfloat16, "half": torch.float16}


def type_of(hip, name):
    return {"float": hip.FLOAT, "bfloat16": hip.BFLOAT16, "half": hip.HALF}[name]


def close(got, want, factor=1.0):
    got = got.cpu()
    m = want.abs().amax(-1, keepdim=True)
    tol = torch.finfo(got.dtype).eps / 2 * want.abs() * (1 + 2.0 ** -10) + 24 * 2.0 ** -24 * m * factor + torch.finfo(got.dtype).tiny * 2.0 ** -10
    off = (got.double() - want).abs() - tol
    assert bool((off <= 0).all()), (float(off.max()), off.argmax())


def rows(tokens, heads, d, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(tokens, heads, d, generator=g).to(dtype)


CASES = [  # tokens, q heads, kv heads, d, rotary_dim, interleaved, norm
    (1, 32, 8, 128, 128, False, True), (1, 1, 1, 2, 2, False, True), (3, 5, 3, 80, 32, True, False), (65, 12, 12, 64, 64, True, True), (17, 3, 1, 96, 48, False, True),
    (9, 8, 2, 256, 256, False, True), (5, 7, 7, 254, 250, False, True), (4, 2, 2, 72, 20, False, True), (4, 2, 2, 72, 20, True, True), (6, 4, 4, 64, 0, False, True),
    (6, 4, 4, 64, 0, False, False), (2, 3, 2, 10, 6, True, True), (700, 9, 3, 128, 64, False, True), (11, 2, 1, 40, 40, False, False), (33, 16, 2, 192, 64, True, True)]


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("tokens,hq,hk,d,r,interleaved,norm", CASES)
def test_norm_rope(hip, dev, name, tokens, hq, hk, d, r, interleaved, norm):
    dtype = TYPES[name]
    q, k = rows(tokens, hq, d, dtype, 1), rows(tokens, hk, d, dtype, 2) * 3
    wq, wk = (1 + 0.2 * torch.randn(2, d, generator=torch.Generator().manual_seed(3))) if norm else (None, None)
    pos = torch.arange(tokens, dtype=torch.int32) * 37 - 5
    pos[-1] = 1000003
    freqs, factor = hip.rope_frequencies(r, 10000.0, hip.ROPE_YARN, 4.0, 64.0, 1.0, 32.0) if r else ([], 1.0)
    freqs = torch.tensor(freqs, dtype=torch.float64)
    p = hip.heads_params(type_of(hip, name), d, hq, hk, rotary_dim=r, interleaved=interleaved, eps=1e-6, attention_factor=factor)
    qd, kd, qo, ko = q.to(dev), k.to(dev), torch.full_like(q, 7, device=dev), torch.full_like(k, 7, device=dev)
    up = lambda x: None if x is None else x.to(dev)
    hip.qk_norm_rope(p, tokens, qd, kd, up(wq), up(wk), pos.to(dev), freqs.to(dev), qo, ko)
    torch.cuda.synchronize()
    for got, x, w in ((qo, q, wq), (ko, k, wk)):
        close(got, ref.norm_rope(x, w, 1e-6, pos, freqs, r, interleaved, factor), max(1.0, factor))
    # one tensor alone and in place gives the same bits
    hip.qk_norm_rope(p, tokens, None, kd, None, up(wk), pos.to(dev), freqs.to(dev), None, kd)
    torch.cuda.synchronize()
    assert torch.equal(kd.cpu(), ko.cpu())


@pytest.mark.parametrize("name", list(TYPES))
def test_norm_rope_of_slices(hip, dev, name):
    """Heads of packed rows, of [heads, tokens, d] tensors, of rows at odd addresses and strides; what lies between stays."""
    dtype, tokens, hq, hk, d = TYPES[name], 21, 6, 2, 64
    freqs, _ = hip.rope_frequencies(d, 10000.0)
    freqs = torch.tensor(freqs, dtype=torch.float64)
    pos = torch.arange(tokens, dtype=torch.int32)
    q, k = rows(tokens, hq, d, dtype, 5), rows(tokens, hk, d, dtype, 6)
    want = [ref.norm_rope(x, None, 0.0, pos, freqs, d, False, 1.0) for x in (q, k)]
    for lead, between in ((0, 0), (16, 16), (4, 4), (1, 3)):
        width = (hq + hk) * (d + between)
        flat = torch.full((lead + tokens * width,), 9.0, dtype=dtype, device=dev)
        heads = flat[lead:].view(tokens, hq + hk, d + between)[..., :d]
        heads[:, :hq], heads[:, hq:] = q.to(dev), k.to(dev)
        out = torch.full((hq + hk, tokens, d), 9.0, dtype=dtype, device=dev)     # head major
        st = (width, d + between)
        p = hip.heads_params(type_of(hip, name), d, hq, hk, rotary_dim=d, q_strides=st, k_strides=st, q_out_strides=(d, tokens * d), k_out_strides=(d, tokens * d))
        hip.qk_norm_rope(p, tokens, heads[:, :hq], heads[:, hq:], None, None, pos.to(dev), freqs.to(dev), out[:hq], out[hq:])
        q2 = hip.heads_params(type_of(hip, name), d, hq, hk, rotary_dim=d, q_strides=st, q_out_strides=st)
        torch.cuda.synchronize()
        close(out[:hq].transpose(0, 1), want[0])
        close(out[hq:].transpose(0, 1), want[1])
        before = flat.clone()
        hip.qk_norm_rope(q2, tokens, heads, None, None, None, pos.to(dev), freqs.to(dev), heads, None)
        torch.cuda.synchronize()
        assert torch.equal(heads[:, :hq], out[:hq].transpose(0, 1))
        heads[:, :hq] = before[lead:].view(tokens, hq + hk, d + between)[:, :hq, :d]
        assert torch.equal(flat, before)     # nothing else was written


def test_norm_of_zeros_and_extremes(hip, dev):
    d = 64
    x = torch.zeros(4, 1, d)
    x[1] = 1e-30
    x[2] = 1e15
    x[3, 0, 5] = math.nan
    p = hip.heads_params(hip.FLOAT, d, 1, 1, eps=1e-6)
    out = torch.empty(4, 1, d, device=dev)
    hip.qk_norm_rope(p, 4, x.to(dev), None, torch.ones(d, device=dev), None, None, None, out, None)
    torch.cuda.synchronize()
    out = out.cpu()
    assert torch.equal(out[0], torch.zeros(1, d)) and torch.isnan(out[3]).all()
    close(out[1], ref.norm_rope(x[1:2], torch.ones(d), 1e-6, None, None, 0, False, 1.0)[0])
    close(out[2], ref.norm_rope(x[2:3], torch.ones(d), 1e-6, None, None, 0, False, 1.0)[0])


def append(hip, dev, name, q, k, v, wq, wk, pos, freqs, r, interleaved, factor, slots, geometry, cache):
    tokens, hq, d = q.shape
    p = hip.heads_params(type_of(hip, name), d, hq, k.shape[1], rotary_dim=r, interleaved=interleaved, eps=1e-6, attention_factor=factor)
    up = lambda x: None if x is None else x.to(dev)
    qo = torch.empty_like(q, device=dev)
    hip.kv4_append(p, geometry, tokens, q.to(dev), k.to(dev), v.to(dev), up(wq), up(wk), pos.to(dev), freqs.to(dev), slots.to(dev), qo, cache)
    torch.cuda.synchronize()
    return qo


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("tokens,hq,hk,d,r,interleaved,norm,page", [
    (1, 32, 8, 128, 128, False, True, 16), (70, 4, 2, 64, 64, True, True, 32), (33, 3, 3, 80, 32, True, False, 16), (19, 5, 5, 72, 20, False, True, 64),
    (40, 2, 1, 256, 256, False, True, 128), (21, 6, 2, 200, 96, False, False, 256), (600, 8, 8, 128, 64, False, True, 16), (5, 1, 1, 8, 8, True, True, 16),
    (9, 3, 1, 40, 6, False, True, 16), (6, 4, 4, 64, 0, False, True, 16)])
def test_append(hip, dev, name, tokens, hq, hk, d, r, interleaved, norm, page):
    dtype = TYPES[name]
    q, k, v = rows(tokens, hq, d, dtype, 1), rows(tokens, hk, d, dtype, 2), rows(tokens, hk, d, dtype, 3)
    v[0] = 0.25                                    # one value: scale 0
    if tokens > 4:
        v[1, :, 0], v[2, 0, 3], k[3, 0, 1] = 1e5 if name != "half" else 65504.0, math.nan, math.nan
        v[4] = (torch.arange(d) % 16).to(dtype)    # every code, ties
    wq, wk = (1 + 0.2 * torch.randn(2, d, generator=torch.Generator().manual_seed(4))) if norm else (None, None)
    pos = (torch.arange(tokens) + 901234).to(torch.int32)
    pos[0] = 0
    freqs, factor = hip.rope_frequencies(r, 500000.0) if r else ([], 1.0)
    freqs = torch.tensor(freqs, dtype=torch.float64)
    pages = -(-tokens // page) + 2
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(5))[:tokens]
    if tokens > 8:
        slots[6], slots[7], slots[8] = -1, pages * page, 1 << 50      # no place in the cache
    geometry = hip.kv4_cache(d, hk, page, pages)
    g = torch.Generator().manual_seed(6)
    start = torch.randint(0, 256, (pages, hip.kv4_page_bytes(geometry)), dtype=torch.uint8, generator=g)
    cache = start.to(dev)
    qo = append(hip, dev, name, q, k, v, wq, wk, pos, freqs, r, interleaved, factor, slots, geometry, cache)
    close(qo, ref.norm_rope(q, wq, 1e-6, pos, freqs, r, interleaved, factor))
    # the cache byte by byte: what was put there, and all else as it was
    kept = [i for i in range(tokens) if 0 <= int(slots[i]) < pages * page]
    content = ref.Cache(pages, hk, d, page, range(0))
    for which, x in ((0, ref.norm_rope(k, wk, 1e-6, pos, freqs, r, interleaved, factor)), (1, v.double())):
        code, scale, offset = ref.quantize(x)
        for i in kept:
            content.code[which, slots[i]], content.scale[which, slots[i]], content.offset[which, slots[i]] = code[i], scale[i, :, 0], offset[i, :, 0]
    want, got = content.pack(), cache.cpu().view(pages, hk, -1)
    written = torch.zeros_like(want)
    dp = ref.padded(d)
    for i in kept:
        n, t = divmod(int(slots[i]), page)
        blk = written[n]
        blk[:, t * dp // 2:(t + 1) * dp // 2] = 1
        for w in range(dp // 8):
            at = page * dp // 2 + (((t // 4) * (dp // 8) + w) * 4 + t % 4) * 4
            blk[:, at:at + 4] = 1
        for base in (page * dp, page * dp + 4 * page):
            at = base + t // 4 * 16 + t % 4 * 2
            blk[:, at:at + 2] = blk[:, at + 8:at + 10] = 1
    same = got == torch.where(written.bool(), want, start.view(pages, hk, -1))
    if not bool(same.all()):   # NaN parameters may have any payload
        par = (torch.arange(want.shape[-1]) >= page * dp)[None, None] & written.bool()
        nan = torch.isnan(torch.where(par, want, torch.zeros_like(want)).view(torch.float16)) & torch.isnan(torch.where(par, got, torch.zeros_like(got)).view(torch.float16))
        same = same | nan.repeat_interleave(2, -1)
    assert bool(same.all()), torch.nonzero(~same)[:10]
    # and read back as values, zeros for the slots that are none
    for out_name, out_type in TYPES.items():
        ko, vo = (torch.full((tokens, hk, d), 7, dtype=out_type, device=dev) for _ in range(2))
        hip.kv4_gather(geometry, type_of(hip, out_name), tokens, cache, slots.to(dev), ko, vo)
        torch.cuda.synchronize()
        for got, vals in ((ko, content.k), (vo, content.v)):
            want = torch.zeros(tokens, hk, d, dtype=torch.float64)
            for i in kept:
                want[i] = vals[slots[i]]
            want = want.float().to(out_type)
            assert torch.equal(torch.isnan(got.cpu()), torch.isnan(want)) and torch.equal(torch.nan_to_num(got.cpu().float()), torch.nan_to_num(want.float()))
    only = torch.full((tokens, hk, d), 7, device=dev)
    hip.kv4_gather(geometry, hip.FLOAT, tokens, cache, slots.to(dev), None, only)
    torch.cuda.synchronize()
    assert torch.equal(torch.nan_to_num(only.cpu()), torch.nan_to_num(vo.cpu().float())) or out_type != torch.float32


def test_append_saturates_infinities(hip, dev):
    d, geometry = 64, hip.kv4_cache(64, 1, 16, 1)
    v = torch.zeros(3, 1, d)
    v[0, 0, 0], v[0, 0, 1], v[1, 0, 2], v[2] = math.inf, -math.inf, 3e38, -math.inf
    cache = torch.zeros(1, hip.kv4_page_bytes(geometry), dtype=torch.uint8, device=dev)
    p = hip.heads_params(hip.FLOAT, d, 1, 1)
    slots = torch.arange(3, device=dev)
    hip.kv4_append(p, geometry, 3, None, v.to(dev), v.to(dev), None, None, None, None, slots, None, cache)
    ko, vo = torch.empty(3, 1, d, device=dev), torch.empty(3, 1, d, device=dev)
    hip.kv4_gather(geometry, hip.FLOAT, 3, cache, slots, ko, vo)
    torch.cuda.synchronize()
    want = ref.values(*ref.quantize(v.double())).float()
    assert torch.equal(ko.cpu(), want) and torch.equal(vo.cpu(), want) and bool(torch.isfinite(want).all())


def test_append_beyond_32_bits(hip, dev):
    """Slots at both ends of a cache of 5 GiB."""
    d, hk, page = 128, 8, 256
    per_page = hip.kv4_page_bytes(hip.kv4_cache(d, hk, page, 1))
    pages = (5 << 30) // per_page
    geometry = hip.kv4_cache(d, hk, page, pages)
    cache = torch.empty(pages * per_page, dtype=torch.uint8, device=dev)
    k = rows(4, hk, d, torch.bfloat16, 7)
    slots = torch.tensor([0, pages * page - 1, pages * page // 2, (1 << 32) // (per_page // page) + 3])
    p = hip.heads_params(hip.BFLOAT16, d, 1, hk)
    hip.kv4_append(p, geometry, 4, None, k.to(dev), k.to(dev), None, None, None, None, slots.to(dev), None, cache)
    ko, vo = torch.empty(4, hk, d, device=dev), torch.empty(4, hk, d, device=dev)
    hip.kv4_gather(geometry, hip.FLOAT, 4, cache, slots.to(dev), ko, vo)
    torch.cuda.synchronize()
    want = ref.values(*ref.quantize(k.double())).float()
    assert torch.equal(ko.cpu(), want) and torch.equal(vo.cpu(), want)


@pytest.mark.parametrize("tokens", [1500, 9001])
def test_many_tokens_are_cut_as_few_are(hip, dev, tokens):
    """More passes than wavefronts: shares that begin and end inside a token, queries in a launch of their own; the same bits as by few tokens a call."""
    hq, hk, d, pages = 20, 4, 64, tokens // 16 + 8
    x = rows(tokens, hq + 2 * hk, d, torch.bfloat16, 9).to(dev)
    freqs = torch.tensor(hip.rope_frequencies(d, 10000.0)[0], dtype=torch.float64, device=dev)
    pos = torch.arange(tokens, dtype=torch.int32, device=dev) * 3
    w = torch.rand(d, device=dev) + 0.5
    st = (x.stride(0), d)
    p = hip.heads_params(hip.BFLOAT16, d, hq, hk, rotary_dim=d, eps=1e-5, q_strides=st, k_strides=st, v_strides=st)
    geometry = hip.kv4_cache(d, hk, 16, pages)
    one, many = (torch.zeros(pages, hip.kv4_page_bytes(geometry), dtype=torch.uint8, device=dev) for _ in range(2))
    q1, q2 = torch.empty(tokens, hq, d, dtype=torch.bfloat16, device=dev), torch.empty(tokens, hq, d, dtype=torch.bfloat16, device=dev)
    slots = torch.arange(tokens, device=dev) + 50
    hip.kv4_append(p, geometry, tokens, x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:], w, w, pos, freqs, slots, q1, many)
    for i in range(0, tokens, 100):
        y = x[i:i + 100]
        hip.kv4_append(p, geometry, len(y), y[:, :hq], y[:, hq:hq + hk], y[:, hq + hk:], w, w, pos[i:], freqs, slots[i:], q2[i:], one)
    torch.cuda.synchronize()
    assert torch.equal(one, many)
    assert torch.equal(q1, q2)
    k1, k2 = torch.empty(tokens, hk, d, dtype=torch.bfloat16, device=dev), torch.empty(tokens, hk, d, dtype=torch.bfloat16, device=dev)
    q3 = torch.empty_like(q1)
    hip.qk_norm_rope(p, tokens, x[:, :hq], x[:, hq:], w, w, pos, freqs, q3, k1)
    for i in range(0, tokens, 100):
        hip.qk_norm_rope(p, min(100, tokens - i), x[i:i + 100, :hq], x[i:i + 100, hq:], w, w, pos[i:], freqs, q2[i:], k2[i:])
    torch.cuda.synchronize()
    assert torch.equal(q3, q2) and torch.equal(k1, k2)


def test_gather_of_more_values_than_a_launch_has(hip, dev):
    """2^31 dwords of codes and some more: the launches' first and last rows, and those where one ends, are what calls of their own read."""
    hk, d = 65535, 8
    geometry = hip.kv4_cache(d, hk, 16, 1)
    tokens = (1 << 31) // hk + 3
    if torch.cuda.mem_get_info()[0] < tokens * hk * d * 2 + (4 << 30):
        pytest.skip("memory for the rows")
    g = torch.Generator(device=dev).manual_seed(1)
    cache = torch.randint(0, 60, (hip.kv4_page_bytes(geometry),), dtype=torch.uint8, device=dev, generator=g)
    slots = torch.arange(tokens, device=dev) * 5 % 16
    out = torch.full((tokens, hk, d), 7, dtype=torch.half, device=dev)
    hip.kv4_gather(geometry, hip.HALF, tokens, cache, slots, out, None)
    once = torch.empty(16, hk, d, dtype=torch.half, device=dev)
    hip.kv4_gather(geometry, hip.HALF, 16, cache, torch.arange(16, device=dev), once, None)
    torch.cuda.synchronize()
    for i in (0, 1, tokens // 2, tokens - 6, tokens - 5, tokens - 4, tokens - 3, tokens - 2, tokens - 1):
        assert torch.equal(out[i], once[i * 5 % 16]), i


def test_replayed_graph_reads_positions_and_slots_anew(hip, dev):
    tokens, hq, hk, d = 7, 4, 2, 64
    geometry = hip.kv4_cache(d, hk, 16, 4)
    cache = torch.zeros(4, hip.kv4_page_bytes(geometry), dtype=torch.uint8, device=dev)
    freqs = torch.tensor(hip.rope_frequencies(d, 10000.0)[0], dtype=torch.float64, device=dev)
    x = torch.zeros(tokens, hq + 2 * hk, d, dtype=torch.half, device=dev)
    pos, slots = torch.zeros(tokens, dtype=torch.int32, device=dev), torch.full((tokens,), -1, device=dev)
    st = (x.stride(0), d)
    p = hip.heads_params(hip.HALF, d, hq, hk, rotary_dim=d, q_strides=st, k_strides=st, v_strides=st)
    qo, ko, vo = torch.empty(tokens, hq, d, dtype=torch.half, device=dev), torch.empty(tokens, hk, d, device=dev), torch.empty(tokens, hk, d, device=dev)

    def step(stream, cache, qo, ko, vo):
        hip.kv4_append(p, geometry, tokens, x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:], None, None, pos, freqs, slots, qo, cache, stream)
        hip.kv4_gather(geometry, hip.FLOAT, tokens, cache, slots, ko, vo, stream)

    step(0, cache, qo, ko, vo)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph, stream=side):
        step(torch.cuda.current_stream().cuda_stream, cache, qo, ko, vo)
    eager = [torch.zeros_like(t) for t in (cache, qo, ko, vo)]
    for i in range(4):
        x.copy_(rows(tokens, hq + 2 * hk, d, torch.half, 20 + i))
        pos.copy_(torch.arange(tokens) + 100 * i)
        slots.copy_(torch.randperm(64, generator=torch.Generator().manual_seed(i))[:tokens] - (1 if i == 2 else 0))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        step(0, *eager)
        torch.cuda.synchronize()
        for a, b in zip((cache, qo, ko, vo), eager):
            assert torch.equal(a, b), i
