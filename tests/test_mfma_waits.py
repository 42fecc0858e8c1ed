"""check_mfma_waits.py, which the build runs over the kernels with inline-assembly MFMAs: it finds a result that is touched too early, on either side of
a branch, accepts enough wait states, and finds nothing in the objects that are built."""
import importlib.util
import os
import shutil

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "spatialthinker_amd", "csrc")


@pytest.fixture(scope="module")
def check():
    spec = importlib.util.spec_from_file_location("check_mfma_waits", os.path.join(CSRC, "check_mfma_waits.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


MFMA = ("v_mfma_f32_16x16x32_bf16", " a[252:255], v[98:101], v[94:97], a[252:255]")


def listing(*ins):
    """(operation, operands[, index of the branch target]) -> what functions() gives: 4 bytes per instruction."""
    return [(4 * i, t[0], t[1], 4 * t[2] if len(t) > 2 else None) for i, t in enumerate(ins)]


@pytest.mark.parametrize("between,found", [
    ([], True),
    ([("s_nop", " 6")], True),                                     # 7 states
    ([("s_nop", " 7")], False),                                    # 8
    ([("s_mov_b32", " s0, s1")] * 7, True),
    ([("s_mov_b32", " s0, s1")] * 8, False),
    ([("v_mfma_f32_16x16x32_bf16", " a[0:3], v[0:3], v[4:7], a[0:3]")] * 1, True),       # 4
    ([("v_mfma_f32_16x16x32_bf16", " a[0:3], v[0:3], v[4:7], a[0:3]")] * 2, False),
])
def test_a_result_read_too_early_is_found(check, between, found):
    code = listing(MFMA, *between, ("v_accvgpr_read_b32", " v5, a255"), ("s_endpgm", ""))
    assert bool(check.early(code)) is found


def test_both_sides_of_a_branch_are_followed(check):
    taken = listing(MFMA, ("s_cbranch_scc1", " 4", 4), ("s_nop", " 7"), ("s_endpgm", ""), ("global_store_dwordx4", " v[0:1], a[252:255], off"), ("s_endpgm", ""))
    not_taken = listing(MFMA, ("s_cbranch_scc1", " 3", 3), ("v_accvgpr_mov_b32", " a1, a254"), ("s_nop", " 7"), ("s_endpgm", ""))
    loop = listing(MFMA, ("s_cbranch_scc1", " 0", 0), ("s_nop", " 7"), ("v_accvgpr_read_b32", " v5, a255"), ("s_endpgm", ""))
    assert check.early(taken) and check.early(not_taken) and not check.early(loop)


def test_another_mfma_may_follow_and_other_registers_do_not_matter(check):
    assert not check.early(listing(MFMA, MFMA, ("s_nop", " 7"), ("v_accvgpr_read_b32", " v5, a255"), ("s_endpgm", "")))
    assert not check.early(listing(MFMA, ("v_accvgpr_read_b32", " v252, a251"), ("v_add_u32_e32", " v255, v254, v253"), ("s_endpgm", "")))
    assert check.early(listing(MFMA, ("v_accvgpr_write_b32", " a253, v1"), ("s_endpgm", "")))          # overwriting it counts too


def test_the_built_kernels_have_their_waits(check):
    objs = [os.path.join(CSRC, n) for n in ("gemm_asm4.o", "vocab_head.o")]
    if not all(os.path.exists(o) for o in objs) or not shutil.which(os.path.join(check.LLVM, "llvm-objdump")):
        pytest.skip("no built objects or no llvm-objdump here")
    seen = check.functions(objs[1])
    assert sum(any(op.startswith("v_mfma") for _, op, _, _ in code) for code in seen.values()) >= 10
    assert check.main(objs) == 0


def test_a_machine_without_objdump_builds_and_says_what_was_not_checked(check, monkeypatch, capsys, tmp_path):
    monkeypatch.setattr(check, "LLVM", str(tmp_path))
    monkeypatch.setenv("PATH", str(tmp_path))
    assert check.main([str(tmp_path / "any.o")]) == 0
    err = capsys.readouterr().err
    assert "llvm-objdump" in err and str(tmp_path) in err and "not checked" in err


def test_an_objdump_on_the_path_will_do(check, monkeypatch, tmp_path):
    tool = tmp_path / "llvm-objdump"
    tool.write_text("#!/bin/sh\nexit 0\n")
    tool.chmod(0o755)
    monkeypatch.setattr(check, "LLVM", str(tmp_path / "nothing"))
    monkeypatch.setenv("PATH", str(tmp_path))
    assert check.objdump() == str(tool)
