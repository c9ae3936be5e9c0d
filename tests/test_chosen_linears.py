"""The operators whose rows choose their weights, without a GPU: prototypes, structures, sizes, refusals."""
import ctypes as C
import math
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "itexhip.h")
ENTRIES = ["route", "group_rows", "experts_up", "experts_down", "adapters"]


def test_prototypes_match_the_header(hip):
    text = open(HEADER).read()
    kind = {"int": C.c_int, "int64_t": C.c_int64, "float": C.c_float}
    assert sorted(hip._CHOSEN) == sorted(ENTRIES)
    for name in ENTRIES:
        args = re.search(r"int itexhip_%s\(([^;]*)\);" % name, text).group(1)
        assert tuple(hip._CHOSEN[name].argtypes) == tuple(C.c_void_p if "*" in a else kind[a.split()[0]] for a in args.split(",")), name
        assert callable(getattr(hip._call, name))


def test_structures_match_the_header(hip, tmp_path):
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "itexhip.h"\nint main(void) { printf("%zu %zu %zu %zu %zu %zu\\n", sizeof(itexhip_route_params), '
                   "sizeof(itexhip_experts_params), sizeof(itexhip_adapters_params), offsetof(itexhip_route_params, logits_stride), "
                   "offsetof(itexhip_experts_params, out_stride), offsetof(itexhip_adapters_params, out_stride)); return 0; }\n")
    subprocess.run(["gcc", "-I", os.path.dirname(HEADER), str(src), "-o", str(tmp_path / "sizes")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "sizes")], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [C.sizeof(hip.RouteParams), C.sizeof(hip.ExpertsParams), C.sizeof(hip.AdaptersParams), hip.RouteParams.logits_stride.offset,
                   hip.ExpertsParams.out_stride.offset, hip.AdaptersParams.out_stride.offset]


ROUTE = dict(type="HALF", experts=64, top_k=4)


@pytest.mark.parametrize("change,match", [
    (dict(type="QINT8"), "type is"), (dict(experts=0), "experts"), (dict(experts=1025), "experts"), (dict(top_k=0), "top_k"), (dict(top_k=33), "top_k"), (dict(experts=3), "top_k"),
    (dict(score=2), "score"), (dict(groups=0), "groups"), (dict(groups=65, experts=65), "groups"), (dict(groups=5), "groups"), (dict(groups=8, top_groups=9), "top_groups"),
    (dict(top_groups=0), "top_groups"), (dict(top_groups=2), "top_groups"), (dict(groups=8, top_groups=1, top_k=9), "top_k"), (dict(group_best=0), "group_best"),
    (dict(group_best=3), "group_best"), (dict(groups=64, group_best=2, top_groups=4), "group_best"), (dict(scale=math.nan), "scale"), (dict(scale=math.inf), "scale"),
    (dict(logits_stride=-1), "logits_stride"), (dict(logits_stride=1 << 31), "logits_stride")])
def test_route_params_that_are_none(hip, change, match):
    kw = {**ROUTE, **change}
    p = hip.route_params(getattr(hip, kw.pop("type")), **kw)
    with pytest.raises(hip.ItexHipError, match=match) as e:
        hip.route(p, 1, 64, None, 64, 64)
    assert e.value.code == hip.INVALID_ARGUMENT


def test_route_refuses(hip):
    p = hip.route_params(hip.HALF, 64, 4)
    for args, match in [((-1, 64, None, 64, 64), "tokens"), ((1 << 30, 64, None, 64, 64), "tokens"), ((1, None, None, 64, 64), "null"), ((1, 64, None, None, 64), "null"),
                        ((1, 64, None, 64, None), "null"), ((1, 65, None, 64, 64), "aligned"), ((1, 64, 66, 64, 64), "aligned"), ((1, 64, None, 66, 64), "aligned"),
                        ((1, 64, None, 64, 66), "aligned")]:
        with pytest.raises(hip.ItexHipError, match=match):
            hip.route(p, *args)
    hip.route(p, 0, None, None, None, None)


def test_group_rows_refuses(hip):
    for n, groups, match in [(-1, 4, "rows are"), (1 << 30, 4, "rows are"), (4, 0, "groups"), (4, 1025, "groups")]:
        with pytest.raises(hip.ItexHipError, match=match):
            hip.group_rows(n, groups, 64, 64, 64, 64)
        with pytest.raises(hip.ItexHipError, match=match):
            hip.group_rows_workspace(n, groups)
    for args, match in [((None, 64, 64, 64), "null"), ((64, None, 64, 64), "null"), ((64, 64, None, 64), "null"), ((64, 64, 64, None), "null"), ((66, 64, 64, 64), "aligned"),
                        ((64, 66, 64, 64), "aligned"), ((64, 64, 66, 64), "aligned"), ((64, 64, 64, 72), "aligned")]:
        with pytest.raises(hip.ItexHipError, match=match):
            hip.group_rows(4, 4, *args)
    with pytest.raises(hip.ItexHipError, match="null"):
        hip.group_rows(0, 4, None, None, None, None)     # offsets are written


EXPERTS = dict(type="BFLOAT16", experts=8, top_k=2, tokens=5, hidden=64, inner=96)


@pytest.mark.parametrize("change,match", [
    (dict(type="QINT32"), "type is"), (dict(experts=0), "experts"), (dict(experts=1025), "experts"), (dict(top_k=0), "top_k"), (dict(top_k=33), "top_k"),
    (dict(tokens=-1), "tokens"), (dict(tokens=1 << 29), "tokens"), (dict(hidden=0), "hidden"), (dict(hidden=65537), "hidden"), (dict(inner=0), "inner"), (dict(inner=65537), "inner"),
    (dict(activation=3), "activation"), (dict(activation=99), "activation"), (dict(x_stride=63), "stride"), (dict(addend_stride=63), "stride"), (dict(out_stride=1 << 31), "stride")])
def test_experts_params_that_are_none(hip, change, match):
    kw = {**EXPERTS, **change}
    p = hip.experts_params(getattr(hip, kw.pop("type")), **kw)
    for call in (lambda: hip.experts_workspace(p), lambda: hip.experts_up(p, 64, 64, 64, 64, 64, 64, 64), lambda: hip.experts_down(p, *([64] * 10))):
        with pytest.raises(hip.ItexHipError, match=match) as e:
            call()
        assert e.value.code == hip.INVALID_ARGUMENT


def test_experts_refuse(hip):
    kw = dict(EXPERTS)
    p = hip.experts_params(getattr(hip, kw.pop("type")), **kw)
    for at in range(7):
        args = [64] * 7
        args[at] = None
        with pytest.raises(hip.ItexHipError, match="null"):
            hip.experts_up(p, *args)
    for at, bad in ((0, 65), (1, 66), (2, 66), (3, 72), (4, 66), (5, 65), (6, 72)):
        args = [64] * 7
        args[at] = bad
        with pytest.raises(hip.ItexHipError, match="aligned"):
            hip.experts_up(p, *args)
    for at in (0, 1, 2, 3, 4, 5, 6, 8, 9):
        args = [64] * 10
        args[at] = None
        with pytest.raises(hip.ItexHipError, match="null"):
            hip.experts_down(p, *args)
    for at, bad in ((0, 65), (1, 66), (2, 66), (3, 66), (4, 72), (5, 66), (6, 66), (7, 65), (8, 65), (9, 72)):
        args = [64] * 10
        args[at] = bad
        with pytest.raises(hip.ItexHipError, match="aligned"):
            hip.experts_down(p, *args)
    other = hip.experts_params(hip.BFLOAT16, **{**{k: v for k, v in EXPERTS.items() if k != "type"}, "addend_stride": 80})
    with pytest.raises(hip.ItexHipError, match="in place"):
        hip.experts_down(other, *([64] * 10))
    empty = hip.experts_params(hip.HALF, **{k: v for k, v in {**EXPERTS, "tokens": 0}.items() if k != "type"})
    hip.experts_up(empty, *([None] * 7))
    hip.experts_down(empty, *([None] * 10))


def test_a_workspace_serves_fewer_tokens(hip):
    for hidden, inner in ((64, 4096), (4096, 64), (770, 1000)):
        sizes = [hip.experts_workspace(hip.experts_params(hip.HALF, 8, 2, t, hidden, inner)) for t in (0, 1, 2, 63, 64, 65, 4096)]
        assert sizes == sorted(sizes) and sizes[0] > 0
        assert sizes[-1] >= 4096 * 2 * (hidden * 4 + inner)
    sizes = [hip.adapters_workspace(hip.adapters_params(hip.HALF, 8, 16, t, 4096, [128])) for t in (0, 1, 2, 15, 16, 17, 63, 64, 65, 255, 256, 257, 4095, 4096, 8192, 100000)]
    assert sizes == sorted(sizes) and sizes[0] > 0
    for groups in (1, 8, 1024):
        sizes = [hip.group_rows_workspace(n, groups) for n in (0, 1, 1023, 1024, 1025, 65536, 10 ** 6, 10 ** 8)]
        assert sizes == sorted(sizes) and sizes[0] > 0


ADAPTERS = dict(type="FLOAT", adapters=4, rank=16, tokens=5, in_dim=64, slice_ends=[96])


@pytest.mark.parametrize("change,match", [
    (dict(type="QUINT8"), "type is"), (dict(adapters=0), "adapters"), (dict(adapters=1025), "adapters"), (dict(rank=0), "rank"), (dict(rank=12), "rank"), (dict(rank=264), "rank"),
    (dict(tokens=-1), "tokens"), (dict(tokens=1 << 30), "tokens"), (dict(in_dim=0), "in is"), (dict(in_dim=(1 << 20) + 1), "in is"), (dict(slice_ends=[0]), "slice_end"),
    (dict(slice_ends=[64, 64]), "slice_end"), (dict(slice_ends=[64, 32]), "slice_end"), (dict(slice_ends=[(1 << 20) + 1]), "slice_end"), (dict(slice_ends=[1, 2, 3, 4, 5]), "slices"),
    (dict(x_stride=63), "x_stride"), (dict(base_stride=95), "stride"), (dict(out_stride=95), "stride"), (dict(out_stride=1 << 31), "stride")])
def test_adapters_params_that_are_none(hip, change, match):
    kw = {**ADAPTERS, **change}
    p = hip.adapters_params(getattr(hip, kw.pop("type")), **kw)
    for call in (lambda: hip.adapters_workspace(p), lambda: hip.adapters(p, *([64] * 10))):
        with pytest.raises(hip.ItexHipError, match=match) as e:
            call()
        assert e.value.code == hip.INVALID_ARGUMENT


def test_adapters_refuse(hip):
    kw = dict(ADAPTERS)
    p = hip.adapters_params(getattr(hip, kw.pop("type")), **kw)
    for at in (0, 1, 2, 3, 4, 6, 7, 8, 9):
        args = [64] * 10
        args[at] = None
        with pytest.raises(hip.ItexHipError, match="null"):
            hip.adapters(p, *args)
    for at, bad in ((0, 66), (1, 66), (2, 66), (3, 66), (4, 72), (5, 66), (6, 66), (7, 66), (8, 66), (9, 72)):
        args = [64] * 10
        args[at] = bad
        with pytest.raises(hip.ItexHipError, match="aligned"):
            hip.adapters(p, *args)
    other = hip.adapters_params(hip.FLOAT, 4, 16, 5, 64, [96], base_stride=128)
    with pytest.raises(hip.ItexHipError, match="in place"):
        hip.adapters(other, *([64] * 10))
    empty = hip.adapters_params(hip.FLOAT, 4, 16, 0, 64, [96])
    hip.adapters(empty, *([None] * 10))
