"""Attention over the paged 4-bit cache against its statement in 64 bits.

Tolerances.  u = 2^-24.  A score of a head of d dimensions is accumulated in fp32 from operands q_j (64 + code) (16-bit types) or q_j code:
d additions of partial sums up to A, then scale and offset: e = scale_softmax (s_max d u A + 4 u |score|) + what a row's queries
lose as halves, 2^-25 of its largest each (nothing for bfloat16 and half rows of like size): the logarithm's error.  A
probability is off by 2 e (its own and the sum's) plus exponential and sums, 40 u, and, for 16-bit types, by the rounding of
probability times scale to a half, 2^-11, or of a value to a half, 2^-11 of it, in long prompts: out is off by (2 e + 40 u + 2^-10) mass
(2 e + 40 u for float), mass = sum p (|scale code| + |offset|), and by half a step of its type."""
import math

import pytest
import torch

from tests import kv4_reference as ref

pytestmark = pytest.mark.gpu
TYPES = {"float": torch.float32, "bfloat16": torch.bfloat16, "half": torch.float16}
U = 2.0 ** -24


def type_of(hip, name):
    return {"float": hip.FLOAT, "bfloat16": hip.BFLOAT16, "half": hip.HALF}[name]


class Batch:
    """Sequences of (new tokens, tokens) in a cache with pages handed out in random order."""

    def __init__(self, lens, heads, group, d, page, seed, extra=2, q_scale=1.0, **cache):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.group, self.d, self.heads = lens, group, d, heads
        need = [-(-n // page) for _, n in lens]
        pages = sum(need) + extra
        order = torch.randperm(pages, generator=g).tolist()
        self.table, used = [], []
        for (_, n), k in zip(lens, need):
            self.table.append([order.pop() for _ in range(k)])
            used += [self.table[-1][t // page] * page + t % page for t in range(n)]
        self.cache = ref.Cache(pages, heads, d, page, used, seed=seed + 1, **cache)
        self.cu = [0]
        for m, _ in lens:
            self.cu.append(self.cu[-1] + m)
        self.q = torch.randn(self.cu[-1], heads * group, d, generator=g) * q_scale

    def table_tensor(self, width=None):
        width = max(1, max(len(t) for t in self.table)) if width is None else width
        out = torch.full((len(self.table), width), -1, dtype=torch.int32)
        for i, t in enumerate(self.table):
            out[i, :len(t)] = torch.tensor(t[:width], dtype=torch.int32)
        return out


def attend(hip, dev, name, batch, causal=True, window=0, rows_behind=3, scale=None, max_q=None, q=None):
    dtype, d, hq = TYPES[name], batch.d, batch.heads * batch.group
    scale = d ** -0.5 if scale is None else scale
    total = batch.cu[-1] + rows_behind
    q = batch.q.to(dtype) if q is None else q
    qd = torch.full((total, hq, d), 5.0, dtype=dtype, device=dev)
    qd[:batch.cu[-1]] = q.to(dev)
    table = batch.table_tensor().to(dev)
    geometry = hip.kv4_cache(d, batch.heads, batch.cache.p, batch.cache.pages)
    p = hip.kv4_attention_params(type_of(hip, name), hq, d, len(batch.lens), max(m for m, _ in batch.lens) if max_q is None else max_q, total, scale, table.shape[1],
                                 causal=causal, window=window)
    ws = torch.full((hip.kv4_attention_workspace(p, geometry),), 0xff, dtype=torch.uint8, device=dev)     # contents irrelevant: NaN
    out, lse = torch.full((total, hq, d), 3.0, dtype=dtype, device=dev), torch.full((total, hq), 3.0, device=dev)
    args = (qd, batch.cache.pack().to(dev), table, torch.tensor(batch.cu, dtype=torch.int32, device=dev), torch.tensor([n for _, n in batch.lens], dtype=torch.int32, device=dev))
    hip.kv4_attention(p, geometry, *args, ws, out, lse)
    torch.cuda.synchronize()
    again = torch.empty_like(out)
    hip.kv4_attention(p, geometry, *args, ws, again)
    torch.cuda.synchronize()
    rows = batch.cu[-1]
    assert torch.equal(again[:rows].view(torch.uint8), out[:rows].view(torch.uint8))               # equal calls, equal bits, with or without lse
    assert bool((out[rows:] == 3.0).all()) and bool((lse[rows:] == 3.0).all())                      # rows behind the last sequence
    return out[:rows].cpu(), lse[:rows].cpu(), q


@pytest.fixture(params=[None, 100000], ids=["", "rows_alone"])
def max_q(request):
    """Of 100000 rows a sequence there are tiles for all CUs: the kernels that divide rows alone run, whatever the sequences then have."""
    return request.param


def check(out, lse, q, batch, causal=True, window=0, scale=None):
    d = batch.d
    scale = d ** -0.5 if scale is None else scale
    want, want_lse, mass = ref.attention(q, batch.cache, batch.table, batch.cu, [n for _, n in batch.lens], scale, causal, window)
    qf = q.double()
    lead = (qf.abs().sum(-1) * 15 + qf.cumsum(-1).abs().amax(-1) * 2 * (72 if out.dtype != torch.float32 else 8))   # A
    scales = batch.cache.scale[torch.isfinite(batch.cache.scale) & (batch.cache.scale.abs() < 60000)]     # (stale places hold more)
    s_max = float(scales.abs().max()) if scales.numel() else 0.0
    score = scale * s_max * 9 * qf.abs().sum(-1) + scale * qf.abs().sum(-1) * 4
    e = scale * s_max * d * U * lead + 4 * U * score + scale * d * 2.0 ** -25 * qf.abs().amax(-1) * s_max * 8
    tol_lse = e + 8 * U * want_lse.abs().nan_to_num(posinf=0) + 40 * U
    empty = torch.isinf(want_lse)
    assert torch.equal(torch.isinf(lse.double()), empty) and bool((lse[empty] < 0).all())
    seen = ~empty & ~torch.isnan(want_lse)
    assert torch.equal(torch.isnan(lse), torch.isnan(want_lse))
    off = ((lse.double() - want_lse).abs() - tol_lse)[seen]
    assert off.numel() == 0 or float(off.max()) <= 0, float(off.max())
    rounding = 2.0 ** -10 if out.dtype != torch.float32 else 0.0
    tol = torch.finfo(out.dtype).eps / 2 * want.abs() * (1 + 2.0 ** -8) + ((2 * e + 40 * U + rounding) * mass)[..., None] + torch.finfo(out.dtype).tiny
    assert torch.equal(torch.isnan(out), torch.isnan(want))
    off = torch.where(torch.isnan(want), torch.zeros_like(want), (out.double() - want).abs() - tol)
    assert off.numel() == 0 or float(off.max()) <= 0, (float(off.max()), int(off.argmax()))
    assert bool((out[empty] == 0).all())


SINGLE = [(1, n) for n in (1, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129, 300)]


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("heads,group,d,page", [(2, 4, 128, 16), (3, 1, 64, 32), (1, 7, 80, 64), (2, 8, 96, 16), (1, 12, 256, 128), (2, 3, 8, 16), (1, 16, 200, 256), (4, 2, 72, 16)])
def test_single_tokens(hip, dev, name, heads, group, d, page):
    batch = Batch(SINGLE, heads, group, d, page, 1)
    check(*attend(hip, dev, name, batch), batch)


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("window", [1, 16, 33, 128, 1000])
def test_single_tokens_with_a_window(hip, dev, name, window):
    batch = Batch(SINGLE, 2, 4, 64, 16, 2)
    check(*attend(hip, dev, name, batch, window=window), batch, window=window)


RAGGED = [(3, 40), (1, 1), (5, 5), (0, 33), (2, 129), (7, 200), (4, 17), (1, 64)]


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("heads,group,d,page,window", [(2, 4, 128, 16, 0), (1, 8, 64, 32, 0), (2, 1, 80, 16, 20), (1, 9, 256, 64, 0), (1, 3, 128, 16, 7), (1, 5, 64, 16, 0)])
@pytest.mark.parametrize("causal", [True, False])
def test_several_tokens(hip, dev, max_q, name, heads, group, d, page, window, causal):
    """1 to 63 rows a sequence and kv head: the split kernels in one tile and several."""
    batch = Batch(RAGGED, heads, group, d, page, 3)
    check(*attend(hip, dev, name, batch, max_q=max_q, causal=causal, window=window), batch, causal=causal, window=window)


PROMPTS = [(70, 70), (1, 90), (33, 150), (0, 10), (129, 129), (64, 64), (40, 41)]


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("heads,group,d,page,window,causal", [(2, 2, 128, 16, 0, True), (1, 4, 64, 32, 0, True), (1, 1, 80, 16, 0, True), (1, 3, 256, 64, 0, True), (1, 2, 128, 16, 30, True),
                                                              (1, 2, 64, 64, 0, False), (1, 2, 200, 16, 50, True), (2, 1, 128, 128, 65, False), (1, 5, 8, 16, 0, True)])
def test_prompts(hip, dev, max_q, name, heads, group, d, page, window, causal):
    batch = Batch(PROMPTS, heads, group, d, page, 4)
    check(*attend(hip, dev, name, batch, max_q=max_q, causal=causal, window=window), batch, causal=causal, window=window)


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("heads,group,d,page,window,causal", [(2, 4, 128, 16, 0, True), (1, 2, 64, 64, 0, False), (1, 4, 256, 32, 0, True), (2, 3, 80, 16, 300, True)])
def test_chunks_behind_long_contexts(hip, dev, max_q, name, heads, group, d, page, window, causal):
    """Hundreds of rows of few sequences: the tokens are divided among workgroups."""
    batch = Batch([(100, 2000), (150, 700), (0, 5), (3, 1500)], heads, group, d, page, 15)
    check(*attend(hip, dev, name, batch, max_q=max_q, causal=causal, window=window), batch, causal=causal, window=window)


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("q_rows", [1, 9, 80])
def test_rows_that_see_nothing(hip, dev, max_q, name, q_rows):
    """More new tokens than tokens, sequences without any, none of them: 0 and lse -inf."""
    batch = Batch([(q_rows, 0), (q_rows, q_rows // 2), (1, 0), (q_rows, q_rows + 3), (0, 0)], 2, 2, 64, 16, 5)
    check(*attend(hip, dev, name, batch, max_q=max_q), batch)
    check(*attend(hip, dev, name, batch, max_q=max_q, causal=False), batch, causal=False)
    batch = Batch([(q_rows, 0)], 1, 1, 128, 16, 5)
    check(*attend(hip, dev, name, batch, max_q=max_q), batch)


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("lens", [[(1, 100), (1, 60)], [(4, 100), (2, 60)], [(80, 100), (1, 60)]])
def test_nan_reaches_only_the_rows_that_see_it(hip, dev, max_q, name, lens):
    for which in (0, 1):
        batch = Batch(lens, 2, 2, 64, 16, 6)
        first, second = batch.table[0], batch.table[1]
        slot = first[98 // 16] * 16 + 98 % 16       # the first sequence's last token but one
        batch.cache.scale[which, slot, 1] = batch.cache.offset[which, slot, 1] = math.nan
        early = second[3 // 16] * 16 + 3
        batch.cache.scale[which, early, 0] = batch.cache.offset[which, early, 0] = math.nan
        out, lse, q = attend(hip, dev, name, batch, max_q=max_q)
        n = lens[0][0]
        assert bool(torch.isnan(out[:n, 2:]).any()) and not bool(torch.isnan(out[:n, :2]).any())
        want, want_lse, _ = ref.attention(q, batch.cache, batch.table, batch.cu, [100, 60], 64 ** -0.5)
        if which == 1:
            want_lse = torch.where(torch.isnan(want).any(-1), torch.nan, want_lse)   # a NaN value makes its rows' sums NaN, lse too
            batch_lse = torch.where(torch.isnan(out).any(-1), torch.nan, lse)
            assert torch.equal(torch.isnan(batch_lse), torch.isnan(want_lse))
        else:
            assert torch.equal(torch.isnan(lse), torch.isnan(want_lse))
        assert torch.equal(torch.isnan(out), torch.isnan(want))
        fine = ~torch.isnan(want)
        assert float((out.double() - want)[fine].abs().max()) < 0.02


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("lens", [[(1, 200)], [(6, 200)], [(90, 200)]])
def test_pages_outside_the_cache_are_not_seen(hip, dev, max_q, name, lens):
    batch = Batch(lens, 1, 2, 128, 32, 7)
    batch.table[0][1] = -1
    batch.table[0][3] = batch.cache.pages
    batch.table[0][4] = 2 ** 31 - 1
    check(*attend(hip, dev, name, batch, max_q=max_q), batch)


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("lens", [[(1, 70), (1, 300)], [(5, 70), (3, 300)], [(90, 100), (70, 300)]])
def test_lengths_beyond_the_table_and_rows_beyond_the_bounds(hip, dev, name, lens):
    batch = Batch(lens, 1, 2, 64, 16, 8)
    dtype, hq, d = TYPES[name], 2, 64
    width = len(batch.table[0])
    table = batch.table_tensor(width).to(dev)
    geometry = hip.kv4_cache(d, 1, 16, batch.cache.pages)
    total = batch.cu[-1]
    q = batch.q.to(dtype)
    cut = [(m, min(n, width * 16)) for m, n in lens]
    want, want_lse, _ = ref.attention(q, batch.cache, [t[:width] for t in batch.table], batch.cu, [n for _, n in cut], d ** -0.5)
    p = hip.kv4_attention_params(type_of(hip, name), hq, d, 2, max(m for m, _ in lens), total, d ** -0.5, width)
    ws = torch.empty(hip.kv4_attention_workspace(p, geometry), dtype=torch.uint8, device=dev)
    out = torch.full((total, hq, d), 3.0, dtype=dtype, device=dev)
    cu = torch.tensor(batch.cu, dtype=torch.int32, device=dev)
    kv = torch.tensor([n for _, n in lens], dtype=torch.int32, device=dev)
    pages = batch.cache.pack().to(dev)
    hip.kv4_attention(p, geometry, q.to(dev), pages, table, cu, kv, ws, out)
    torch.cuda.synchronize()
    assert float((out.cpu().double() - want).abs().max()) < 0.02
    # a sequence said to be longer than max_q_len, a last row beyond total_q, a negative length, a falling row list: no access out of bounds
    few = hip.kv4_attention_params(type_of(hip, name), hq, d, 2, 1, total - 1, d ** -0.5, width)
    for cu_bad, kv_bad in (([0, total + 100, total + 200], [70, 70]), ([-5, 1, 2], [-7, 1 << 30]), ([2, 0, 1], [50, 50]), ([1 << 30, 0, 1 << 30], [70, 70])):
        out.fill_(3.0)
        hip.kv4_attention(few, geometry, q.to(dev), pages, table, torch.tensor(cu_bad, dtype=torch.int32, device=dev), torch.tensor(kv_bad, dtype=torch.int32, device=dev), ws, out)
        torch.cuda.synchronize()
        assert bool((out[total - 1:] == 3.0).all())


@pytest.mark.parametrize("name", list(TYPES))
def test_many_sequences(hip, dev, name):
    """More sequences than threads in a workgroup: the scan over them in pieces; most of them without rows."""
    lens = [(1 if i % 3 else 0, 1 + (i * 37) % 70) for i in range(600)]
    batch = Batch(lens, 1, 2, 64, 16, 9)
    check(*attend(hip, dev, name, batch), batch)


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("heads,group,d", [(1, 4, 128), (2, 1, 64), (1, 2, 256)])
def test_long_contexts_shared_by_many_workgroups(hip, dev, name, heads, group, d):
    batch = Batch([(1, 5000), (1, 3), (2, 2999)], heads, group, d, 64, 10)
    check(*attend(hip, dev, name, batch), batch)


@pytest.mark.parametrize("name", ["bfloat16", "half", "float"])
def test_rising_scores_and_scales(hip, dev, max_q, name):
    """Maxima that grow step by step, values whose scales grow over 2^20, rows of very different size: the sums are rescaled."""
    batch = Batch([(1, 400), (3, 400), (100, 400)], 1, 2, 64, 16, 11)
    for b in range(3):
        for t in range(400):
            slot = batch.table[b][t // 16] * 16 + t % 16
            batch.cache.scale[0, slot] = torch.tensor(0.002 * t + 0.01).half().double()
            batch.cache.scale[1, slot] = torch.tensor(2.0 ** (-18 + t // 20)).double()
            batch.cache.offset[1, slot] = torch.tensor(2.0 ** (-16 + t // 20)).double()
    batch.q *= torch.logspace(-3, 1, batch.cu[-1])[:, None, None]
    check(*attend(hip, dev, name, batch, max_q=max_q), batch)


@pytest.mark.parametrize("name", ["bfloat16", "half"])
def test_queries_beyond_halves(hip, dev, max_q, name):
    """bfloat16 queries far outside half's range, zero queries, tiny softmax scales."""
    batch = Batch([(1, 50), (2, 50), (70, 90)], 1, 2, 64, 16, 12)
    big = 1e30 if name == "bfloat16" else 6e4
    batch.q[0] *= big / 4
    batch.q[1] = 0
    batch.q[5] *= 1e-30 if name == "bfloat16" else 1e-6
    q = batch.q.to(TYPES[name])
    for scale in (1.0 / big, 1e-38, 0.125 if name == "half" else 1e-30):
        out, lse, _ = attend(hip, dev, name, batch, max_q=max_q, scale=scale, q=q)
        want, want_lse, mass = ref.attention(q, batch.cache, batch.table, batch.cu, [n for _, n in batch.lens], scale)
        assert bool(torch.isfinite(out).all())
        if scale != 0.125:
            assert float(((out.double() - want).abs() / mass[..., None]).max()) < 2.0 ** -7 and float((lse - want_lse).abs().max()) < 1e-3


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("lens", [[(1, 100), (1, 30)], [(6, 100), (3, 30)], [(70, 100), (2, 30)]])
def test_strides(hip, dev, name, lens):
    """Queries as slices of packed rows, head major, at odd strides; outputs likewise."""
    batch = Batch(lens, 2, 3, 64, 16, 13)
    dtype, hq, d, total = TYPES[name], 6, 64, batch.cu[-1]
    base, base_lse, q = attend(hip, dev, name, batch)
    geometry = hip.kv4_cache(d, 2, 16, batch.cache.pages)
    table = batch.table_tensor().to(dev)
    rest = (batch.cache.pack().to(dev), table, torch.tensor(batch.cu, dtype=torch.int32, device=dev), torch.tensor([n for _, n in lens], dtype=torch.int32, device=dev))
    for lead, row, head, orow, ohead in ((0, 10 * d, d, hq * d, d), (0, d, total * d, d, total * d), (1, hq * (d + 3), d + 3, hq * (d + 1), d + 1)):
        size = lead + (total - 1) * max(row, orow) + (hq - 1) * max(head, ohead) + total * d + 64
        qs, os = torch.zeros(size, dtype=dtype, device=dev), torch.full((size,), 3.0, dtype=dtype, device=dev)
        torch.as_strided(qs, (total, hq, d), (row, head, 1), lead).copy_(q.to(dev))
        p = hip.kv4_attention_params(type_of(hip, name), hq, d, 2, max(m for m, _ in lens), total, d ** -0.5, table.shape[1], q_strides=(row, head), out_strides=(orow, ohead))
        ws = torch.empty(hip.kv4_attention_workspace(p, geometry), dtype=torch.uint8, device=dev)
        hip.kv4_attention(p, geometry, qs[lead:], *rest, ws, os[lead:])
        torch.cuda.synchronize()
        view = torch.as_strided(os, (total, hq, d), (orow, ohead, 1), lead)
        assert torch.equal(view.cpu(), base)
        view.fill_(3.0)
        assert bool((os == 3.0).all())


@pytest.mark.parametrize("lens", [[(1, 200), (1, 30)], [(6, 100), (3, 30)], [(90, 100), (2, 30)]])
def test_replayed_graphs_and_two_streams(hip, dev, lens):
    """A captured step reads lengths, tables and rows anew; two graphs that take turns share a workspace; two streams at once have one each."""
    batch = Batch(lens, 2, 2, 128, 16, 14)
    hq, d, total = 4, 128, batch.cu[-1]
    geometry = hip.kv4_cache(d, 2, 16, batch.cache.pages)
    table = batch.table_tensor().to(dev)
    pages = batch.cache.pack().to(dev)
    p = hip.kv4_attention_params(hip.BFLOAT16, hq, d, 2, max(m for m, _ in lens), total, d ** -0.5, table.shape[1])
    size = hip.kv4_attention_workspace(p, geometry)
    q = torch.zeros(total, hq, d, dtype=torch.bfloat16, device=dev)
    cu, kv = torch.tensor(batch.cu, dtype=torch.int32, device=dev), torch.ones(2, dtype=torch.int32, device=dev)
    ws = torch.empty(size, dtype=torch.uint8, device=dev)
    outs = [torch.zeros_like(q) for _ in range(2)]
    step = lambda w, o, st: hip.kv4_attention(p, geometry, q, pages, table, cu, kv, w, o, None, st)
    graphs = []
    for o in outs:
        step(ws, o, 0)
        torch.cuda.synchronize()
        g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(g, stream=side):
            step(ws, o, torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    want, w2 = torch.zeros_like(q), torch.empty(size, dtype=torch.uint8, device=dev)
    for i in range(4):
        q.copy_(torch.randn(total, hq, d, generator=torch.Generator().manual_seed(i)))
        kv.copy_(torch.tensor([max(m, n - 13 * i) for m, n in lens]))
        step(w2, want, 0)
        torch.cuda.synchronize()
        for g, o in zip(graphs, outs):
            o.zero_()
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(o, want), i
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for i in range(20):
        step(ws, outs[0], a.cuda_stream)
        step(w2, outs[1], b.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


def test_cache_beyond_32_bits(hip, dev):
    """A sequence whose pages lie at both ends of 5 GiB."""
    d, heads, page = 128, 2, 16
    per_page = hip.kv4_page_bytes(hip.kv4_cache(d, heads, page, 1))
    pages = (5 << 30) // per_page
    for lens in ([(1, 90)], [(5, 90)], [(80, 90)]):
        batch = Batch(lens, heads, 2, d, page, 15)
        small = batch.cache.pack()
        big = torch.empty(pages, per_page, dtype=torch.uint8, device=dev)
        place = [0, pages - 1, pages // 2, pages - 2, 1, pages - 3]
        for i, n in enumerate(batch.table[0]):
            big[place[i]] = small[n].reshape(-1).to(dev)
        p = hip.kv4_attention_params(hip.HALF, 4, d, 1, lens[0][0], lens[0][0], d ** -0.5, 6)
        geometry = hip.kv4_cache(d, heads, page, pages)
        ws = torch.empty(hip.kv4_attention_workspace(p, geometry), dtype=torch.uint8, device=dev)
        out, lse = torch.empty(lens[0][0], 4, d, dtype=torch.half, device=dev), torch.empty(lens[0][0], 4, device=dev)
        q = batch.q.half()
        hip.kv4_attention(p, geometry, q.to(dev), big, torch.tensor([place], dtype=torch.int32, device=dev), torch.tensor(batch.cu, dtype=torch.int32, device=dev),
                          torch.tensor([90], dtype=torch.int32, device=dev), ws, out, lse)
        torch.cuda.synchronize()
        check(out.cpu(), lse.cpu(), q, batch)
        del big


def test_a_decoder_layer_from_prompt_to_tokens(hip, dev):
    """Rows of a qkv linear -> append -> attention, a prompt and then token by token, as a server runs it: every step's output is that of plain attention over
    the cache's values, and the tokens' rows are those of the whole sequence in one go."""
    hq, hk, d, page, n, tail = 8, 2, 64, 16, 75, 6
    g = torch.Generator().manual_seed(16)
    x = torch.randn(n + tail, hq + 2 * hk, d, generator=g).to(torch.bfloat16).to(dev)
    w = torch.ones(d, device=dev)
    freqs = torch.tensor(hip.rope_frequencies(d, 500000.0)[0], dtype=torch.float64, device=dev)
    st = (x.stride(0), d)
    heads = hip.heads_params(hip.BFLOAT16, d, hq, hk, rotary_dim=d, eps=1e-6, q_strides=st, k_strides=st, v_strides=st)
    geometry = hip.kv4_cache(d, hk, page, 8)
    table = torch.tensor([[5, 0, 7, 2, 3, 6]], dtype=torch.int32, device=dev)
    slot = lambda t: table[0, t // page].long() * page + t % page
    outs = {}
    for chunks in ([n] + [1] * tail, [n + tail], [40, 41]):
        cache = torch.zeros(8, hip.kv4_page_bytes(geometry), dtype=torch.uint8, device=dev)
        done, got = 0, []
        for m in chunks:
            rows, t = x[done:done + m], torch.arange(done, done + m, device=dev)
            q = torch.empty(m, hq, d, dtype=torch.bfloat16, device=dev)
            hip.kv4_append(heads, geometry, m, rows[:, :hq], rows[:, hq:hq + hk], rows[:, hq + hk:], w, w, t.to(torch.int32), freqs, slot(t), q, cache)
            done += m
            p = hip.kv4_attention_params(hip.BFLOAT16, hq, d, 1, m, m, d ** -0.5, 6)
            ws = torch.empty(hip.kv4_attention_workspace(p, geometry), dtype=torch.uint8, device=dev)
            out = torch.empty(m, hq, d, dtype=torch.bfloat16, device=dev)
            hip.kv4_attention(p, geometry, q, cache, table, torch.tensor([0, m], dtype=torch.int32, device=dev), torch.tensor([done], dtype=torch.int32, device=dev), ws, out)
            got.append((q, out))
        ko, vo = torch.empty(done, hk, d, device=dev), torch.empty(done, hk, d, device=dev)
        hip.kv4_gather(geometry, hip.FLOAT, done, cache, slot(torch.arange(done, device=dev)), ko, vo)
        torch.cuda.synchronize()
        q, out = (torch.cat(v).cpu().double() for v in zip(*got))
        k, v = ko.cpu().double().repeat_interleave(hq // hk, 1), vo.cpu().double().repeat_interleave(hq // hk, 1)
        z = torch.matmul(q.transpose(0, 1), k.permute(1, 2, 0)) * d ** -0.5
        z = z.masked_fill(torch.ones(done, done, dtype=torch.bool).triu(1), -math.inf)
        want = torch.matmul(z.softmax(-1), v.transpose(0, 1)).transpose(0, 1)
        assert float((out - want).abs().max()) <= 2.0 ** -8 * float(want.abs().max()) + 2.0 ** -9 * float(v.abs().max())
        outs[tuple(chunks)] = (cache.cpu(), q, out)
    first = outs[(n + tail,)]
    for cache, q, out in outs.values():
        assert torch.equal(cache, first[0]) and torch.equal(q, first[1])      # the cache does not depend on how the tokens came
        assert float((out - first[2]).abs().max()) <= 2.0 ** -7 * float(first[2].abs().max())


@pytest.mark.skipif("torch.cuda.device_count() < 2")
def test_another_device(hip):
    d, geometry = 64, hip.kv4_cache(64, 1, 16, 2)
    other = torch.device("cuda:1")
    with torch.cuda.device(other):
        batch = Batch([(1, 20)], 1, 2, d, 16, 17)
        check(*attend(hip, other, "half", batch), batch)


def placed(batch, b, t):
    """The slot of a sequence's token."""
    return batch.table[b][t // batch.cache.p] * batch.cache.p + t % batch.cache.p


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("d", [64, 128, 256])
def test_a_workspace_serves_smaller_calls(hip, dev, name, d):
    """A workspace of the largest call and what lies behind it, with calls of fewer rows, sequences and pages: prompts, chunks, single tokens."""
    most = hip.kv4_attention_params(type_of(hip, name), 4, d, 3, 300, 1000, d ** -0.5, 60)
    for lens in ([(1, 900), (1, 30), (1, 950)], [(4, 700), (9, 30)], [(30, 900)], [(300, 300), (2, 40)], [(70, 900)]):
        batch = Batch(lens, 2, 2, d, 16, 23)
        table = batch.table_tensor().to(dev)
        geometry = hip.kv4_cache(d, 2, 16, batch.cache.pages)
        size = hip.kv4_attention_workspace(most, geometry)
        held = torch.full((size + 4096,), 0xa5, dtype=torch.uint8, device=dev)
        out, lse, q = attend(hip, dev, name, batch)
        p = hip.kv4_attention_params(type_of(hip, name), 4, d, len(lens), max(m for m, _ in lens), batch.cu[-1], d ** -0.5, table.shape[1])
        assert hip.kv4_attention_workspace(p, geometry) <= size
        again, lse2 = torch.empty_like(out, device=dev), torch.empty_like(lse, device=dev)
        hip.kv4_attention(p, geometry, q.to(dev), batch.cache.pack().to(dev), table, torch.tensor(batch.cu, dtype=torch.int32, device=dev),
                          torch.tensor([n for _, n in lens], dtype=torch.int32, device=dev), held, again, lse2)
        torch.cuda.synchronize()
        assert torch.equal(again.cpu(), out) and torch.equal(lse2.cpu(), lse)
        assert bool((held[size:] == 0xa5).all())


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("lens", [[(1, 200), (1, 60)], [(6, 200), (3, 60)], [(90, 200), (70, 90)]])
def test_saturated_values(hip, dev, max_q, name, lens, d):
    """Rows of values with an element of 65504 or more: the codes of the largest stand for up to 65536, beyond what a half holds."""
    batch = Batch(lens, 2, 2, d, 16, 18)
    rows = torch.full((3, d), 0.5, dtype=torch.float64)
    rows[0, 3], rows[1, 5], rows[2, 1], rows[2, 2] = 65504.0, math.inf, math.inf, -math.inf
    rows[:, 7] = 0.0
    code, scale, offset = ref.quantize(rows)
    assert float(ref.values(code, scale, offset).max()) == 65536.0 and float(ref.values(code, scale, offset)[0].max()) == 65520.0
    for b, (m, n) in enumerate(lens):
        for head in range(2):
            for i, t in enumerate((n - 2 if head else 9, 20 + head, n - m // 2 - 1)):    # some rows see them, all do, some of a tile do not
                slot = placed(batch, b, t)
                batch.cache.code[1, slot, head], batch.cache.scale[1, slot, head], batch.cache.offset[1, slot, head] = code[i], scale[i, 0], offset[i, 0]
    out, lse, q = attend(hip, dev, name, batch, max_q=max_q)
    assert bool(torch.isfinite(out).all()) and bool(torch.isfinite(lse).all())
    check(out, lse, q, batch)


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("lens,d", [([(1, 100), (1, 300)], 64), ([(4, 100), (2, 300)], 128), ([(80, 100), (40, 300)], 128), ([(4, 100), (40, 200)], 256), ([(1, 100), (30, 60)], 256)])
def test_values_that_are_not_finite(hip, dev, max_q, name, bad, lens, d):
    """A scale or an offset of a value that is NaN or infinite: rows that see it are NaN in out and lse, whether or not other rows of a step see it too,
    and the others are what they are without it."""
    for which in ("both", "scale", "offset"):
        for b, t in ((0, 98), (0, 3), (1, 3)):                         # seen by the first sequence's last rows; by all rows of one
            batch = Batch(lens, 2, 2, d, 16, 19)
            plain = Batch(lens, 2, 2, d, 16, 19)
            slot = placed(batch, b, t)
            if which != "offset":
                batch.cache.scale[1, slot, 1] = bad
            if which != "scale":
                batch.cache.offset[1, slot, 1] = bad
            out, lse, q = attend(hip, dev, name, batch, max_q=max_q)
            rows, hit = torch.arange(batch.cu[-1]), torch.zeros(batch.cu[-1], 4, dtype=torch.bool)
            m, n = lens[b]
            hit[:, 2:] = ((rows >= batch.cu[b]) & (rows < batch.cu[b + 1]) & (n - m + rows - batch.cu[b] >= t))[:, None]
            assert torch.equal(torch.isnan(lse), hit) and torch.equal(torch.isnan(out), hit[..., None].expand_as(out))
            want, want_lse, mass = ref.attention(q, plain.cache, plain.table, plain.cu, [n for _, n in lens], d ** -0.5)
            out, lse = torch.where(hit[..., None], want.to(out.dtype), out), torch.where(hit, want_lse.float(), lse)
            check(out, lse, q, plain)


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("heads,group,d,window,causal", [(2, 2, 64, 0, True), (1, 4, 128, 0, True), (1, 3, 256, 0, True), (2, 2, 64, 20, True), (1, 3, 128, 9, False)])
@pytest.mark.parametrize("lens,most", [([(8, 100), (1, 60), (5, 5)], 4), ([(120, 170), (3, 60), (70, 70), (80, 50)], 66), ([(8, 100), (3, 2), (6, 90)], 1)])
def test_rows_that_are_not_computed_keep_the_others_positions(hip, dev, name, lens, most, heads, group, d, window, causal):
    """Sequences with more rows than max_q_len, and one with rows beyond total_q: row i of n sits at kv_len - n + i all the same."""
    batch = Batch(lens, heads, group, d, 16, 20)
    dtype, hq = TYPES[name], heads * group
    for total in (batch.cu[-1], batch.cu[-1] - 2):
        q = batch.q.to(dtype)
        table = batch.table_tensor().to(dev)
        geometry = hip.kv4_cache(d, heads, 16, batch.cache.pages)
        for bound in (most, 100000):
            p = hip.kv4_attention_params(type_of(hip, name), hq, d, len(lens), bound, total, d ** -0.5, table.shape[1], causal=causal, window=window)
            ws = torch.empty(hip.kv4_attention_workspace(p, geometry), dtype=torch.uint8, device=dev)
            out, lse = torch.full((batch.cu[-1], hq, d), 3.0, dtype=dtype, device=dev), torch.full((batch.cu[-1], hq), 3.0, device=dev)
            hip.kv4_attention(p, geometry, q.to(dev), batch.cache.pack().to(dev), table, torch.tensor(batch.cu, dtype=torch.int32, device=dev),
                              torch.tensor([n for _, n in lens], dtype=torch.int32, device=dev), ws, out, lse)
            torch.cuda.synchronize()
            out, lse = out.cpu(), lse.cpu()
            rows = torch.arange(batch.cu[-1])
            done = rows < total
            for b, (m, _) in enumerate(lens):
                done &= ~((rows >= batch.cu[b] + bound) & (rows < batch.cu[b + 1]))
            assert int(done.sum()) < len(rows) or bound == 100000
            assert bool((out[~done] == 3.0).all()) and bool((lse[~done] == 3.0).all())
            want, want_lse, _ = ref.attention(q, batch.cache, batch.table, batch.cu, [n for _, n in lens], d ** -0.5, causal, window)
            out[~done], lse[~done] = want[~done].to(dtype), want_lse[~done].float()
            check(out, lse, q, batch, causal=causal, window=window)


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 30])
@pytest.mark.parametrize("q_rows", [5, 9, 80])
def test_windows_beyond_every_length(hip, dev, max_q, name, q_rows, window):
    """Among sequences of more new tokens than tokens, whose first rows sit before position 0."""
    batch = Batch([(q_rows, q_rows // 2), (1, 40), (q_rows, q_rows + 3), (q_rows, 1), (0, 0)], 2, 2, 64, 16, 21)
    for causal in (True, False):
        check(*attend(hip, dev, name, batch, max_q=max_q, causal=causal, window=window), batch, causal=causal, window=window)


@pytest.mark.parametrize("name", list(TYPES))
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("order", ["large first", "large at first", "falling", "large unseen", "large among small", "larger scores of smaller scales", "any"])
def test_falling_scales(hip, dev, max_q, name, d, order):
    """Values whose scales differ by up to 2^30, the large ones without probability in the end: what is left keeps its bits.  Keys' offsets times a sum of
    queries of about 10 / scale order the scores; two tokens have nearly all of the probability, so that no average hides what they lost."""
    lens = [(1, 900), (3, 900), (100, 900)]
    batch = Batch(lens, 1, 2, d, 16, 22, q_scale=0.05)
    batch.q += 10.0 / math.sqrt(d)
    batch.cache.scale[0] = torch.tensor(0.02).half().double()
    g = torch.Generator().manual_seed(24)
    for b, (_, n) in enumerate(lens):
        for t in range(n):
            slot = placed(batch, b, t)
            large = {"large first": t == 5, "large at first": t < 20, "large unseen": t == n - 1, "large among small": t % 8 == 3}.get(order, False)
            scale, low = (4096.0, -4.0) if large else (2.0 ** -18, 0.0)
            if order == "falling":
                scale, low = 2.0 ** max(12 - t // 16, -18), 4.0 * (min(t, 600) / 600 - 1)
            if order == "larger scores of smaller scales":
                scale, low = 2.0 ** ((t * 7) % 24 - 18), -0.1 * ((t * 7) % 24)
            if order == "any":
                scale, low = 2.0 ** float(torch.rand(1, generator=g) * 30 - 18), -4.0 * float(torch.rand(1, generator=g))
            if t in (690, 700):                                      # all rows see them
                scale, low = 2.0 ** -18, 1.93 if t == 690 else 2.0
            batch.cache.scale[1, slot], batch.cache.offset[0, slot], batch.cache.offset[1, slot] = 1.37 * scale, low, 0.0
    batch.cache.offset, batch.cache.scale = batch.cache.offset.half().double(), batch.cache.scale.half().double()
    out, lse, q = attend(hip, dev, name, batch, max_q=max_q)
    want, want_lse, mass = ref.attention(q, batch.cache, batch.table, batch.cu, [n for _, n in lens], d ** -0.5)
    qf, eps, tiny = q.double(), torch.finfo(out.dtype).eps, torch.finfo(out.dtype).tiny
    lead = qf.abs().sum(-1) * 15 + qf.cumsum(-1).abs().amax(-1) * 2 * (72 if name != "float" else 8)
    e = d ** -0.5 * (0.02 * d * U * lead + 4 * U * (0.02 * 9 + 4) * qf.abs().sum(-1) + d * 2.0 ** -25 * qf.abs().amax(-1) * 0.02 * 8)
    assert float(((lse.double() - want_lse).abs() - e - 8 * U * want_lse.abs() - 40 * U).max()) <= 0
    rounding = 2.0 ** -10 if name != "float" else 0.0
    tol = eps / 2 * want.abs() * (1 + 2.0 ** -8) + tiny * eps + ((2 * e + 40 * U + rounding) * mass)[..., None]
    if name == "bfloat16" and max_q:
        # prompts take a probability to a half apart from its value's scale, as 2^9 of the largest so far or more: below 2^-14 it is off by up to 2^-25, that is
        # 2^-34 of the largest, which is at most 1 of the sum: 2^-34 of each value's magnitude
        total = torch.stack([8.0 * batch.cache.scale[1, [placed(batch, b, t) for t in range(n)], 0].sum() for b, (_, n) in enumerate(lens)])
        tol += 2.0 ** -34 * total.repeat_interleave(torch.tensor([m for m, _ in lens]))[:, None, None]
    off = (out.double() - want).abs() - tol
    assert float(off.max()) <= 0, (float(off.max()), float(((out.double() - want).abs() / mass[..., None]).max()))


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("lens", [[(1, 300)], [(5, 300), (2, 90)], [(90, 300)]])
def test_zeros_add_nothing_in_float(hip, dev, max_q, lens, d):
    """Keys that are zero (codes of 8, no offset) beside large queries: every product is zero exactly, the sums are counts of tokens."""
    batch = Batch(lens, 2, 2, d, 16, 25, q_scale=100.0)
    batch.cache.code[0], batch.cache.scale[0], batch.cache.offset[0] = 8, 4.0, 0.0
    out, lse, q = attend(hip, dev, "float", batch, max_q=max_q)
    want, want_lse, mass = ref.attention(q, batch.cache, batch.table, batch.cu, [n for _, n in lens], d ** -0.5)
    assert float(((lse.double() - want_lse).abs() - 8 * U * want_lse.abs() - 40 * U).max()) <= 0
    assert float(((out.double() - want).abs() - 2.0 ** -24 * want.abs() - 40 * U * mass[..., None]).max()) <= 0
