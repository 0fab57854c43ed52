"""No kernel spills a register where a part of the lanes only would store it.

hipcc was seen to end a branch of the lanes with a spill of an address in front of the instruction that brings the other
lanes back: those reloaded what they had not stored, and wrote there.  tda_amd.isa_check looks for such places in every kernel's assembly.
CPU only (hipcc cross-compiles); the synthetic snippets pin the scanner itself."""
import os

import pytest

from tda_amd import build, isa_check


def _spills(body: str) -> list:
    return isa_check.masked_spills(isa_check._functions("_Z1kv:\n" + body + "\n\ts_endpgm\n.Lfunc_end0:\n")["_Z1kv"])


BRANCH = """
\ts_and_saveexec_b64 s[6:7], vcc
\ts_cbranch_execz .LBB0_2
\tglobal_load_dwordx4 v[2:5], v[6:7], off
.LBB0_2:
"""


def test_scanner_flags_a_spill_before_the_lanes_are_back():
    assert _spills(BRANCH + """\tv_mov_b32_e32 v211, v202
\tscratch_store_dwordx2 off, v[98:99], off
\ts_or_b64 exec, exec, s[6:7]
\tscratch_store_dword off, v8, off offset:8""") == [(".LBB0_2", "scratch_store_dwordx2 off, v[98:99], off")]


def test_scanner_accepts_spills_of_all_lanes_and_of_a_branch():
    assert _spills(BRANCH + """\ts_or_b64 exec, exec, s[6:7]
\tscratch_store_dwordx2 off, v[98:99], off""") == []
    assert _spills(BRANCH + """\ts_or_saveexec_b64 s[4:5], s[4:5]
\tscratch_store_dword off, v8, off
\ts_xor_b64 exec, exec, s[4:5]
\ts_or_b64 exec, exec, s[4:5]""") == []
    # no branch leads here: a block that the lanes run through
    assert _spills(""".LBB0_3:
\tscratch_store_dword off, v8, off
\ts_or_b64 exec, exec, s[4:5]""") == []


def test_scanner_flags_spills_to_accumulator_registers():
    assert _spills(BRANCH + """\tv_accvgpr_write_b32 a12, v98
\tv_accvgpr_write_b32 a13, 0
\tv_accvgpr_write_b32 a14, s3
\tv_writelane_b32 v255, s34, 2
\tv_accvgpr_read_b32 v4, a9
\ts_or_b64 exec, exec, s[6:7]
\tv_accvgpr_write_b32 a15, v99""") == [(".LBB0_2", "v_accvgpr_write_b32 a12, v98")]


@pytest.mark.parametrize("back", ["s_or_b64 exec, exec, s[6:7]", "s_or_saveexec_b64 s[4:5], s[6:7]", "s_mov_b64 exec, s[6:7]"])
@pytest.mark.parametrize("spill", ["scratch_store_dword off, v98, off", "v_accvgpr_write_b32 a12, v98"])
def test_scanner_knows_each_way_back(back, spill):
    assert _spills(BRANCH + f"\t{spill}\n\t{back}") == [(".LBB0_2", spill)]
    assert _spills(BRANCH + f"\t{back}\n\t{spill}") == []


def test_kernels_are_read_to_their_end():
    body = isa_check._functions("_Z1kv:\n\ts_cbranch_scc1 .LBB0_2\n\ts_endpgm\n.LBB0_2:\n\tv_mov_b32_e32 v3, 0\n\ts_endpgm\n.Lfunc_end0:\n\tv_nop\n")["_Z1kv"]
    assert [kind for kind, _ in body] == ["ins", "end", "label", "ins", "end"]


@pytest.mark.skipif(not os.path.exists(build.HIPCC), reason="hipcc not available")
def test_kernels_have_no_spills_under_a_mask():
    assert isa_check.check_spills() == {}
