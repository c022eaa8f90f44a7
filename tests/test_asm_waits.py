"""The build's check of scalar registers that a vector instruction wrote (asmcheck.check_sgpr_waits) follows the
control flow: five wait states before a vector-memory instruction reads them, on every path."""
import importlib.util
import re
import sys
from pathlib import Path

import pytest

PKG = Path(__file__).resolve().parent.parent / "im-not-llm_amd"


def _module(name):
    spec = importlib.util.spec_from_file_location(f"{name}_flow", PKG / f"{name}.py")
    m = importlib.util.module_from_spec(spec)
    sys.modules[spec.name] = m
    spec.loader.exec_module(m)
    return m


@pytest.fixture(scope="module")
def waits():
    check = _module("asmcheck").check_sgpr_waits

    def run(*lines):
        return check("k:\n" + "".join(l + "\n" if l.endswith(":") else f"\t{l}\n" for l in lines) + "\ts_endpgm\n.Lfunc_end0:\n")
    return run


WRITE = "v_readfirstlane_b32 s4, v3"
LOAD = "buffer_load_dwordx4 v3, s[4:7], 0 offen lds"
FIVE = [f"s_mov_b32 s{i}, 0" for i in range(20, 25)]


def test_a_taken_branch_skips_the_states_between(waits):
    bad = waits(WRITE, "s_cbranch_scc1 .LBB0_2", *FIVE, ".LBB0_2:", LOAD)
    assert len(bad) == 1 and bad[0].registers == ["s4"] and "wait states" in str(bad[0])
    assert not waits(WRITE, "s_cbranch_scc1 .LBB0_2", *FIVE, ".LBB0_2:", "s_nop 3", LOAD)
    # a scalar write in the skipped block does not end the wait
    assert len(waits(WRITE, "s_cbranch_scc1 .LBB0_2", "s_mov_b32 s4, 0", ".LBB0_2:", LOAD)) == 1
    assert not waits(WRITE, "s_mov_b32 s4, 0", "s_cbranch_scc1 .LBB0_2", *FIVE, ".LBB0_2:", LOAD)
    # and what cannot be reached is no path
    assert not waits(WRITE, "s_branch .LBB0_2", LOAD, ".LBB0_2:", "s_nop 4", LOAD)


def test_the_end_of_a_loop_stands_before_its_head(waits):
    loop = [".LBB0_1:", LOAD, *FIVE]
    assert len(waits(*loop, WRITE, "s_cbranch_scc1 .LBB0_1")) == 1
    assert not waits(*loop, WRITE, *FIVE[:4], "s_cbranch_scc1 .LBB0_1")
    assert not waits(".LBB0_1:", "s_nop 4", LOAD, WRITE, "s_cbranch_scc1 .LBB0_1")


def test_registers(waits):
    # a compare of scalars and a wait write nothing
    assert len(waits(WRITE, "s_cmp_eq_u32 s4, 0", LOAD)) == 1
    assert len(waits(WRITE, "s_waitcnt vmcnt(0)", LOAD)) == 1
    # carries, the LDS address, offsets
    assert len(waits("v_add_co_u32_e64 v0, s[6:7], v1, v2", LOAD)) == 1
    assert len(waits("v_readfirstlane_b32 m0, v3", LOAD)) == 1
    assert not waits("v_readfirstlane_b32 m0, v3", "buffer_load_dwordx4 v[0:3], v4, s[4:7], 0 offen")
    assert len(waits("v_cmp_lt_u32_e64 s[8:9], v0, v1", "buffer_load_dword v0, v1, s[4:7], s9 offen")) == 1
    assert not waits("v_add_u32_e32 v0, s4, v1", LOAD)
    for states in range(7):
        bad = waits(WRITE, *(f"s_mov_b32 s{30 + i}, 0" for i in range(states)), LOAD)
        assert len(bad) == (states < 5), states


def test_sources_with_asm_loads_are_checked():
    """Every source that issues vector memory operations from inline asm, by itself or by a call of a header's function
    that does, is among those whose listings the build checks."""
    issues = re.compile(r'"[^"\n]*(buffer|global|flat|scratch)_(load|store|atomic)_')
    held = _module("build").NO_SCRATCH
    calls = set()
    for h in (PKG / "csrc").glob("*.hpp"):
        text = h.read_text()
        for m in issues.finditer(text):
            calls.add(re.findall(r"(\w+)\([^;{}]*\)\s*\{", text[:m.start()])[-1])
    assert calls
    found = {s.name for s in (PKG / "csrc").glob("*.hip")
             if issues.search(s.read_text()) or any(re.search(rf"\b{c}\(", s.read_text()) for c in calls)}
    assert "attn_bwd.hip" in found and found <= held, found - held


def test_static_lds_is_found():
    """The kernel of wide heads' dk and dv tells its two stages apart by one bit of an LDS address."""
    build = _module("build")
    text = lambda size, name="attn_bwd_pair_kernel": (f"\t.amdhsa_kernel _Z20{name}ILi256ELb1EEvv\n"
                                                      f"\t\t.amdhsa_group_segment_fixed_size {size}\n")
    build.check_no_static_lds("attn_bwd.hip", text(0) + text(16, "another_kernel"))
    with pytest.raises(RuntimeError, match="static LDS: .*pair_kernel.* .16 bytes"):
        build.check_no_static_lds("attn_bwd.hip", text(0) + text(16))
    with pytest.raises(RuntimeError, match="no static LDS size"):
        build.check_no_static_lds("attn_bwd.hip", text(0, "another_kernel"))
    build.check_no_static_lds("attn_pp.hip", "")
    assert set(build.NO_STATIC_LDS) <= build.NO_SCRATCH
