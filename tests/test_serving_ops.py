"""The operators between a decoder's qkv linear and its output linear, without a GPU: refusals, host-only functions, the binding's
prototypes, the cache's layout."""
import ctypes as C
import math
import os
import re
import subprocess

import pytest
import torch

from tests import kv4_reference as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "itexhip.h")
ENTRIES = ["qk_norm_rope", "kv4_append", "kv4_gather", "kv4_attention"]


def test_prototypes_match_the_header(hip):
    text = open(HEADER).read()
    kind = {"int": C.c_int, "int64_t": C.c_int64, "float": C.c_float, "double": C.c_double}
    assert sorted(hip._SERVING) == sorted(ENTRIES)
    for name in ENTRIES:
        args = re.search(r"int itexhip_%s\(([^;]*)\);" % name, text).group(1)
        assert tuple(hip._SERVING[name].argtypes) == tuple(C.c_void_p if "*" in a else kind[a.split()[0]] for a in args.split(",")), name
        assert callable(getattr(hip._call, name))


def test_structures_match_the_header(hip, tmp_path):
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "itexhip.h"\nint main(void) { printf("%zu %zu %zu %zu %zu\\n", sizeof(itexhip_heads_params), '
                   "sizeof(itexhip_kv4_cache), sizeof(itexhip_kv4_attention_params), offsetof(itexhip_heads_params, q_strides), "
                   "offsetof(itexhip_kv4_attention_params, table_stride)); return 0; }\n")
    subprocess.run(["gcc", "-I", os.path.dirname(HEADER), str(src), "-o", str(tmp_path / "sizes")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "sizes")], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [C.sizeof(hip.HeadsParams), C.sizeof(hip.Kv4Cache), C.sizeof(hip.Kv4AttentionParams), hip.HeadsParams.q_strides.offset,
                   hip.Kv4AttentionParams.table_stride.offset]


@pytest.mark.parametrize("d,heads,page", [(8, 1, 16), (64, 12, 32), (72, 3, 64), (128, 8, 16), (200, 2, 256), (256, 1, 128)])
def test_page_bytes(hip, d, heads, page):
    assert hip.kv4_page_bytes(hip.kv4_cache(d, heads, page, 1)) == heads * page * (ref.padded(d) + 8)


@pytest.mark.parametrize("d,heads,page,pages,match", [(0, 1, 16, 1, "head_dim"), (12, 1, 16, 1, "multiple of 8"), (264, 1, 16, 1, "head_dim"), (64, 0, 16, 1, "kv_heads"),
                                                      (64, 65536, 16, 1, "kv_heads"), (64, 1, 8, 1, "page_size"), (64, 1, 48, 1, "page_size"), (64, 1, 512, 1, "page_size"),
                                                      (64, 1, 16, 0, "num_pages"), (64, 1, 16, 1 << 31, "num_pages")])
def test_geometries_that_are_none(hip, d, heads, page, pages, match):
    c = hip.kv4_cache(d, heads, page, pages)
    p = hip.kv4_attention_params(hip.HALF, max(heads, 1), max(d, 8), 1, 1, 1, 0.125, 4)
    for call in (lambda: hip.kv4_page_bytes(c), lambda: hip.kv4_attention_workspace(p, c), lambda: hip.kv4_gather(c, hip.HALF, 1, 64, 64, 64, 64),
                 lambda: hip.kv4_attention(p, c, 64, 64, 64, 64, 64, 64, 64),
                 lambda: hip.kv4_append(hip.heads_params(hip.HALF, 64, 1, 1), c, 1, None, 64, 64, None, None, None, None, 64, None, 64)):
        with pytest.raises(hip.ItexHipError, match=match) as e:
            call()
        assert e.value.code == hip.INVALID_ARGUMENT


HEADS = dict(type="HALF", head_dim=64, q_heads=4, kv_heads=2, rotary_dim=32)


@pytest.mark.parametrize("change,match", [(dict(type="QINT8"), "type is"), (dict(head_dim=63), "head_dim"), (dict(head_dim=258), "head_dim"), (dict(head_dim=0), "head_dim"),
                                          (dict(rotary_dim=66), "rotary_dim"), (dict(rotary_dim=7), "rotary_dim"), (dict(rotary_dim=-2), "rotary_dim"), (dict(eps=-1.0), "eps"),
                                          (dict(eps=math.nan), "eps"), (dict(attention_factor=math.inf), "attention_factor"), (dict(q_heads=-1), "heads"),
                                          (dict(kv_heads=1 << 16), "heads"), (dict(q_strides=(1 << 41, 64)), "stride"), (dict(k_out_strides=(64, -(1 << 41))), "stride")])
def test_rows_of_heads_that_are_none(hip, change, match):
    kw = {**HEADS, **change}
    p = hip.heads_params(getattr(hip, kw.pop("type")), **kw)
    with pytest.raises(hip.ItexHipError, match=match):
        hip.qk_norm_rope(p, 1, 64, 64, None, None, 64, 64, 64, 64)
    with pytest.raises(hip.ItexHipError, match=match):
        hip.kv4_append(p, hip.kv4_cache(64, 2, 16, 4), 1, None, 64, 64, None, None, 64, 64, 64, None, 64)


def test_norm_rope_refuses(hip):
    p = hip.heads_params(hip.HALF, 64, 4, 2, rotary_dim=32)
    for args, match in [((-1, 64, 64, None, None, 64, 64, 64, 64), "tokens"), ((1 << 31, 64, 64, None, None, 64, 64, 64, 64), "tokens"),
                        ((1, 64, 64, None, None, 64, 64, None, 64), "without its output"), ((1, 64, None, None, None, 64, 64, 64, 64), "without its output"),
                        ((1, 64, 64, None, None, None, 64, 64, 64), "positions and freqs"), ((1, 64, 64, None, None, 64, None, 64, 64), "positions and freqs"),
                        ((1, 65, 64, None, None, 64, 64, 64, 64), "aligned"), ((1, 64, 64, 66, None, 64, 64, 64, 64), "aligned"), ((1, 64, 64, None, None, 66, 64, 64, 64), "aligned"),
                        ((1, 64, 64, None, None, 64, 68, 64, 64), "aligned")]:
        with pytest.raises(hip.ItexHipError, match=match):
            hip.qk_norm_rope(p, *args)
    other = hip.heads_params(hip.HALF, 64, 4, 2, q_strides=(512, 64))
    with pytest.raises(hip.ItexHipError, match="in place"):
        hip.qk_norm_rope(other, 1, 64, None, None, None, None, None, 64, None)
    hip.qk_norm_rope(p, 0, None, None, None, None, None, None, None, None)       # nothing to do
    hip.qk_norm_rope(p, 3, None, None, None, None, 64, 64, None, None)


def test_append_and_gather_refuse(hip):
    p, c = hip.heads_params(hip.HALF, 64, 4, 2, rotary_dim=32), hip.kv4_cache(64, 2, 16, 4)
    ok = dict(tokens=1, q=None, k=64, v=64, q_weight=None, k_weight=None, positions=64, freqs=64, slots=64, q_out=None, cache=64)
    for change, match in [(dict(k=None), "null"), (dict(v=None), "null"), (dict(slots=None), "null"), (dict(cache=None), "null"), (dict(q=64), "without its output"),
                          (dict(q_out=64), "without its output"), (dict(positions=None), "positions and freqs"), (dict(cache=72), "aligned"), (dict(slots=68), "aligned"),
                          (dict(v=65), "aligned"), (dict(tokens=-1), "tokens")]:
        with pytest.raises(hip.ItexHipError, match=match):
            hip.kv4_append(p, c, **{**ok, **change})
    for bad in (hip.kv4_cache(64, 3, 16, 4), hip.kv4_cache(128, 2, 16, 4)):
        with pytest.raises(hip.ItexHipError, match="cache's"):
            hip.kv4_append(p, bad, **ok)
    hip.kv4_append(p, c, **{**ok, "tokens": 0, "k": None, "v": None, "cache": None})
    for args, match in [((hip.QINT8, 1, 64, 64, 64, 64), "type"), ((hip.HALF, -1, 64, 64, 64, 64), "tokens"), ((hip.HALF, 1, None, 64, 64, 64), "null"),
                        ((hip.HALF, 1, 64, None, 64, 64), "null"), ((hip.HALF, 1, 64, 64, 72, 64), "aligned"), ((hip.HALF, 1, 64, 64, 64, 72), "aligned")]:
        with pytest.raises(hip.ItexHipError, match=match):
            hip.kv4_gather(c, *args)
    hip.kv4_gather(c, hip.HALF, 0, None, None, None, None)
    hip.kv4_gather(c, hip.HALF, 5, None, None, None, None)


ATTENTION = dict(type="BFLOAT16", q_heads=8, head_dim=64, num_seqs=2, max_q_len=1, total_q=2, scale=0.125, table_stride=4)


@pytest.mark.parametrize("change,match", [(dict(type="QUINT8"), "type is"), (dict(q_heads=7), "multiple of kv_heads"), (dict(q_heads=0), "multiple of kv_heads"),
                                          (dict(num_seqs=-1), "num_seqs"), (dict(num_seqs=65536), "num_seqs"), (dict(max_q_len=-1), "max_q_len"), (dict(max_q_len=1 << 28), "max_q_len"),
                                          (dict(total_q=1 << 31), "total_q"), (dict(scale=0.0), "scale"), (dict(scale=math.nan), "scale"), (dict(scale=math.inf), "scale"),
                                          (dict(window=-1), "window"), (dict(table_stride=-1), "table_stride"), (dict(table_stride=1 << 27), "table_stride"),
                                          (dict(out_strides=(1 << 41, 64)), "stride")])
def test_attention_params_that_are_none(hip, change, match):
    kw = {**ATTENTION, **change}
    p, c = hip.kv4_attention_params(getattr(hip, kw.pop("type")), **kw), hip.kv4_cache(64, 2, 16, 4)
    with pytest.raises(hip.ItexHipError, match=match):
        hip.kv4_attention_workspace(p, c)
    with pytest.raises(hip.ItexHipError, match=match):
        hip.kv4_attention(p, c, 64, 64, 64, 64, 64, 64, 64)


def test_attention_refuses(hip):
    kw = dict(ATTENTION)
    p, c = hip.kv4_attention_params(getattr(hip, kw.pop("type")), **kw), hip.kv4_cache(64, 2, 16, 4)
    names = ["q", "cache", "block_table", "cu_q", "kv_len", "workspace", "out"]
    for i, name in enumerate(names):
        args = [64] * 7
        args[i] = None
        with pytest.raises(hip.ItexHipError, match="null"):
            hip.kv4_attention(p, c, *args)
    for i, bad in enumerate([65, 72, 66, 66, 66, 72, 65]):
        args = [64] * 7
        args[i] = bad
        with pytest.raises(hip.ItexHipError, match="aligned"):
            hip.kv4_attention(p, c, *args)
    with pytest.raises(hip.ItexHipError, match="aligned"):
        hip.kv4_attention(p, c, *([64] * 7), lse=66)
    for zero in ("num_seqs", "max_q_len", "total_q"):
        hip.kv4_attention(hip.kv4_attention_params(hip.HALF, **{**kw, zero: 0}), c, *([None] * 7))
    assert hip.kv4_attention_workspace(p, c) > 0


def test_other_forms_of_arguments_go_through_the_prototypes(hip):
    import numpy as np
    p, c = hip.heads_params(hip.HALF, 64, 4, 2), hip.kv4_cache(64, 2, 16, 4)
    hip.qk_norm_rope(p, np.int64(0), None, None, None, None, None, None, None, None, None)
    hip.kv4_append(p, c, np.int64(0), None, None, None, None, None, None, None, None, None, None)
    hip.kv4_gather(c, np.int32(hip.HALF), np.int64(0), None, None, None, None)
    with pytest.raises(hip.ItexHipError, match="tokens"):
        hip.kv4_gather(c, hip.HALF, np.int64(-1), None, None, None, None)
    a = hip.kv4_attention_params(hip.HALF, 4, 64, 1, 1, 1, 0.125, 4)
    with pytest.raises(hip.ItexHipError, match="null"):
        hip.kv4_attention(a, c, np.uint64(64), None, None, None, None, None, None)


def frequencies(r, base):
    return [base ** (-2.0 * i / r) / (2.0 * math.pi) for i in range(r // 2)]


def test_frequencies(hip):
    close = lambda a, b: all(abs(x - y) <= 1e-14 * abs(y) for x, y in zip(a, b)) and len(a) == len(b)
    f, m = hip.rope_frequencies(128, 10000.0)
    assert close(f, frequencies(128, 10000.0)) and m == 1.0
    f, m = hip.rope_frequencies(64, 10000.0, hip.ROPE_LINEAR, 4.0)
    assert close(f, [x / 4.0 for x in frequencies(64, 10000.0)]) and m == 1.0
    f, m = hip.rope_frequencies(64, 10000.0, hip.ROPE_NTK, 8.0)
    assert close(f, frequencies(64, 10000.0 * 8.0 ** (64.0 / 62.0))) and m == 1.0
    f, m = hip.rope_frequencies(128, 500000.0, hip.ROPE_LLAMA3, 8.0, 8192.0, 1.0, 4.0)
    plain, want = frequencies(128, 500000.0), []
    for x in plain:
        turns = 8192.0 * x
        want.append(x if turns > 4.0 else x / 8.0 if turns < 1.0 else (1.0 - (turns - 1.0) / 3.0) * x / 8.0 + (turns - 1.0) / 3.0 * x)
    assert close(f, want) and m == 1.0 and f[0] == plain[0] and f[-1] == plain[-1] / 8.0
    f, m = hip.rope_frequencies(128, 10000.0, hip.ROPE_YARN, 16.0, 4096.0, 1.0, 32.0)
    plain = frequencies(128, 10000.0)
    first, last = (128 * math.log(4096.0 / (t * 2.0 * math.pi)) / (2.0 * math.log(10000.0)) for t in (32.0, 1.0))
    first, last = math.floor(first), math.ceil(last)
    want = [x / 16.0 * min(1.0, max(0.0, (i - first) / (last - first))) + x * (1.0 - min(1.0, max(0.0, (i - first) / (last - first)))) for i, x in enumerate(plain)]
    assert close(f, want) and abs(m - (0.1 * math.log(16.0) + 1.0)) < 1e-15
    assert f[0] == plain[0] and abs(f[-1] - plain[-1] / 16.0) <= 1e-15 * f[-1]


@pytest.mark.parametrize("args,match", [((63, 1e4), "rotary_dim"), ((0, 1e4), "rotary_dim"), ((258, 1e4), "rotary_dim"), ((64, 1.0), "base"), ((64, math.inf), "base"),
                                        ((64, 1e4, 9), "scaling"), ((64, 1e4, 1, 0.5), "factor"), ((2, 1e4, 2, 2.0), "NTK"), ((64, 1e4, 3, 8.0, 0.0, 1.0, 4.0), "original_context"),
                                        ((64, 1e4, 4, 8.0, 4096.0, 32.0, 1.0), "low < high")])
def test_frequencies_refuse(hip, args, match):
    with pytest.raises(hip.ItexHipError, match=match):
        hip.rope_frequencies(*args)


def test_layout_is_the_documented_one(tmp_path):
    """csrc/kv4.hpp's offsets against the reference packing: every byte of a block has one owner."""
    src = tmp_path / "offsets.cc"
    src.write_text("""#include <cstdio>
#include <initializer_list>
#include "kv4.hpp"
int main() { for (int dp : {64, 128, 256}) for (int p : {16, 64}) { itexhip::Kv4Block b{p, dp}; std::printf("%d %d %d", dp, p, b.bytes());
for (int t = 0; t < p; ++t) { std::printf(" %d %d %d", b.key_codes(t), b.key_params(t), b.value_params(t)); for (int w = 0; w < dp / 8; ++w) std::printf(" %d", b.value_codes(t, w)); }
std::printf("\\n"); } }
""")
    csrc = os.path.join(ROOT, "intel-extension-for-tensorflow_amd", "csrc")
    subprocess.run(["g++", "-std=c++17", "-I", os.path.dirname(HEADER), "-I", csrc, str(src), "-o", str(tmp_path / "offsets")], check=True)
    for line in subprocess.run([str(tmp_path / "offsets")], check=True, capture_output=True, text=True).stdout.splitlines():
        n = [int(x) for x in line.split()]
        dp, p, size = n[:3]
        assert size == p * (dp + 8)
        owners = [0] * size
        at = 3
        for t in range(p):
            k, kp, vp = n[at:at + 3]
            assert (k, kp, vp) == (t * dp // 2, p * dp + t // 4 * 16 + t % 4 * 2, p * dp + 4 * p + t // 4 * 16 + t % 4 * 2)
            spans = [(k, dp // 2), (kp, 2), (kp + 8, 2), (vp, 2), (vp + 8, 2)]
            for w in range(dp // 8):
                v = n[at + 3 + w]
                assert v == p * dp // 2 + ((t // 4 * (dp // 8) + w) * 4 + t % 4) * 4
                spans.append((v, 4))
            for a, m in spans:
                for i in range(a, a + m):
                    owners[i] += 1
            at += 3 + dp // 8
        assert owners == [1] * size


def test_reference_quantizer_by_hand():
    code, scale, offset = ref.quantize(torch.tensor([[0.0, 15.0, 7.5, 3.0], [2.0, 2.0, 2.0, 2.0]], dtype=torch.float64))
    assert scale.tolist() == [[1.0], [0.0]] and offset.tolist() == [[8.0], [2.0]]
    assert code.tolist() == [[0, 15, 8, 3], [8, 8, 8, 8]]      # (7.5 - 8) / 1 = -0.5 goes to even, 0
    assert ref.values(code, scale, offset).tolist() == [[0.0, 15.0, 8.0, 3.0], [2.0, 2.0, 2.0, 2.0]]


@pytest.mark.parametrize("type", ["FLOAT", "BFLOAT16", "HALF"])
@pytest.mark.parametrize("d,heads,group", [(64, 1, 2), (128, 8, 4), (128, 1, 1), (256, 2, 8), (80, 4, 16)])
def test_a_workspace_serves_smaller_calls(hip, type, d, heads, group):
    """Which kernel takes a call depends on its sizes: a prompt's may need less than a token's."""
    c = hip.kv4_cache(d, heads, 16, 1000)
    size = lambda seqs, rows, pages, **kw: hip.kv4_attention_workspace(
        hip.kv4_attention_params(getattr(hip, type), heads * group, d, seqs, rows, seqs * max(rows, 1), 0.125, pages, **kw), c)
    seqs, rows, pages = (1, 2, 64), (0, 1, 3, 5, 9, 17, 65, 90, 300, 8192, 100000), (0, 1, 19, 300, 8192)
    sizes = {(b, m, n): size(b, m, n) for b in seqs for m in rows for n in pages}
    for b, m, n in sizes:
        assert sizes[b, m, n] == size(b, m, n, window=100) == size(b, m, n, causal=False)
        for b2 in seqs:
            for m2 in rows:
                for n2 in pages:
                    if b2 <= b and m2 <= m and n2 <= n:
                        assert sizes[b2, m2, n2] <= sizes[b, m, n]


@pytest.mark.parametrize("page,stride", [(256, (1 << 56) + 1), (256, 1 << 62), (256, (1 << 22) + 1), (16, 1 << 60), (16, (1 << 63) - 1), (16, (1 << 26) + 1), (128, (1 << 57) + 8)])
def test_tables_beyond_the_bound_whatever_their_product_wraps_to(hip, page, stride):
    c = hip.kv4_cache(64, 2, page, 4)
    p = hip.kv4_attention_params(hip.BFLOAT16, 8, 64, 2, 1, 2, 0.125, stride)
    with pytest.raises(hip.ItexHipError, match="table_stride"):
        hip.kv4_attention_workspace(p, c)
    with pytest.raises(hip.ItexHipError, match="table_stride"):
        hip.kv4_attention(p, c, 64, 64, 64, 64, 64, 64, 64)


@pytest.mark.parametrize("page", [16, 256])
def test_the_widest_table_is_taken(hip, page):
    p = hip.kv4_attention_params(hip.BFLOAT16, 8, 64, 2, 1, 2, 0.125, (1 << 30) // page)
    assert hip.kv4_attention_workspace(p, hip.kv4_cache(64, 2, page, 4)) > 0
