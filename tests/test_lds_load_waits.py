"""Direct loads to LDS written as inline assembly get no hazard wait states from the compiler.  The build checks the device
assembly of the units that have them (csrc/check_asm_hazards.py); here: the checker flags such a load on hand-made assembly, every
unit that can have one is checked, and what the last build left behind is clean."""
import glob
import importlib.util
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "intel-extension-for-tensorflow_amd")
ASM_LOAD = re.compile(r'asm\s+volatile\s*\(\s*"([^"]*global_load_lds[^"]*)"')


def load(path, name):
    spec = importlib.util.spec_from_file_location(name, path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.fixture(scope="module")
def chk():
    return load(os.path.join(PKG, "csrc", "check_asm_hazards.py"), "check_asm_hazards_of_lds_loads")


@pytest.fixture(scope="module")
def build():
    return load(os.path.join(PKG, "build.py"), "itex_amd_build_of_lds_loads")


def flagged(chk, tmp_path, capsys, lines):
    f = tmp_path / "k.s"
    f.write_text("_Z6kernelv:\n" + "".join(l + "\n" if l.startswith((".", "_")) else "\t" + l + "\n" for l in lines))
    n = chk.check_file(str(f))
    return n, capsys.readouterr().out


LOAD = "global_load_lds_dwordx4 v1, s[4:5]"


@pytest.mark.parametrize("between,bad", [([], 1), (["s_nop 0"], 0), (["v_add_f32_e32 v2, v2, v2"], 0)])
def test_a_wait_state_after_m0(chk, tmp_path, capsys, between, bad):
    n, out = flagged(chk, tmp_path, capsys, [";;#ASMSTART", "s_mov_b32 m0, s3"] + between + [LOAD, ";;#ASMEND", "s_endpgm"])
    assert n == bad, out
    assert ("write of m0" in out) == bool(bad)


def test_m0_written_where_a_branch_comes_from(chk, tmp_path, capsys):
    """m0 is written last before a jump: a branch is a wait state, falling through a label is none."""
    n, out = flagged(chk, tmp_path, capsys, ["s_mov_b32 m0, s3", ".LBB0_1:", ";;#ASMSTART", LOAD, ";;#ASMEND", "s_cbranch_scc1 .LBB0_1", "s_endpgm"])
    assert n == 1, out
    n, out = flagged(chk, tmp_path, capsys, ["s_branch .LBB0_2", ".LBB0_1:", ";;#ASMSTART", LOAD, ";;#ASMEND", "s_endpgm", ".LBB0_2:", "s_mov_b32 m0, s3", "s_branch .LBB0_1"])
    assert n == 0, out


@pytest.mark.parametrize("before,bad", [
    (["v_readfirstlane_b32 s4, v3", "s_add_i32 s9, s9, 1", "s_mov_b32 m0, s3", "s_nop 0"], 1), (["v_readfirstlane_b32 s4, v3", "s_nop 3"], 1),
    (["v_readfirstlane_b32 s4, v3", "s_nop 4"], 0), (["v_readfirstlane_b32 s4, v3", "s_nop 1", "v_mov_b32_e32 v9, 0", "s_nop 1"], 0),
    (["v_readfirstlane_b32 s6, v3", "s_mov_b32 s4, s6"], 0), (["v_cmp_lt_u32_e64 s[4:5], v3, v4"], 1), (["v_add_co_u32_e64 v7, s[4:5], v3, v4"], 1),
    (["v_readfirstlane_b32 s5, v3", ".LBB0_1:", "s_nop 3"], 1), (["s_cbranch_scc1 .LBB0_3", "s_nop 4", ".LBB0_3:"], 0),
    (["v_readlane_b32 s5, v3, 4", "s_cbranch_scc1 .LBB0_3", "s_nop 4", ".LBB0_3:"], 1)])
def test_five_wait_states_after_a_vector_instruction_wrote_the_base(chk, tmp_path, capsys, before, bad):
    n, out = flagged(chk, tmp_path, capsys, before + [";;#ASMSTART", LOAD, ";;#ASMEND", "s_endpgm"])
    assert n == bad, out
    assert ("wait state(s) between v_" in out) == bool(bad)


def test_the_compiler_s_own_loads_are_not_looked_at(chk, tmp_path, capsys):
    assert flagged(chk, tmp_path, capsys, ["s_mov_b32 m0, s3", LOAD, "v_readfirstlane_b32 s4, v3", LOAD, "s_endpgm"])[0] == 0


def test_every_unit_with_such_a_load_is_checked(build):
    """They stand in two headers' helpers and in one unit; who calls a helper is checked too."""
    sources = glob.glob(os.path.join(PKG, "csrc", "*.hpp")) + glob.glob(os.path.join(PKG, "csrc", "*.hip"))
    having = sorted(os.path.basename(f) for f in sources if ASM_LOAD.search(open(f).read()))
    assert having == ["experts.hip", "qgemm_common.hpp"]
    calling = [f for f in sources if re.search(r"\blds_dma16\w*(<[^;]*>)?\(", open(f).read())]
    assert sorted(os.path.basename(f) for f in calling) == ["experts.hip", "qgemm_common.hpp", "qgemm_tile.hpp"]
    for f in glob.glob(os.path.join(PKG, "csrc", "*.hip")):
        if ASM_LOAD.search(open(f).read()) or '"qgemm_tile.hpp"' in open(f).read():
            assert build.keeps_assembly(f), os.path.basename(f)
    for f in sources:
        for text in ASM_LOAD.findall(open(f).read()):
            assert re.search(r"m0, [^;]*?\\n\\ts_nop \d+\\n\\tglobal_load_lds", text), (os.path.basename(f), text)


def test_assembly_of_the_last_build_is_clean(chk, build, capsys):
    """(the units of the quantized MatMul's tiles: test_asm_hazards.py)"""
    f = build.device_assembly_of(os.path.join(PKG, "csrc", "experts.hip"))
    if not os.path.exists(f):
        pytest.skip("device assembly not present (the library was not built in this tree)")
    assert "global_load_lds_dwordx4" in open(f).read()
    assert chk.check_file(f) == 0, capsys.readouterr().out
