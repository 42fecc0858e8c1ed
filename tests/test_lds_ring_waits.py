"""Rings of LDS slots that copies fill behind a barrier: in the built code of the vocabulary-head kernels and the GEMM tile every LDS read has returned when its
wave reaches a barrier, so that no copy can overtake it."""
import importlib.util
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "spatialthinker_amd", "csrc")


@pytest.fixture(scope="module")
def check():
    spec = importlib.util.spec_from_file_location("check_mfma_waits", os.path.join(CSRC, "check_mfma_waits.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def pending_reads(code):
    """Addresses of barriers that an LDS read may reach before it has returned (they return in order: lgkmcnt(n) leaves the n youngest)."""
    at = {a: i for i, (a, *_) in enumerate(code)}
    bad = set()
    for i, (_, op, _, _) in enumerate(code):
        if not op.startswith("ds_read"):
            continue
        todo, seen = [(i + 1, 0)], {}
        while todo:
            j, younger = todo.pop()
            while j < len(code) and seen.get(j, younger + 1) > younger:
                seen[j] = younger
                addr, o, args, target = code[j]
                if o == "s_barrier":
                    bad.add("%x" % addr)
                    break
                m = re.search(r"lgkmcnt\((\d+)\)", args) if o == "s_waitcnt" else None
                if m and int(m.group(1)) <= younger:
                    break
                younger += o.startswith("ds_")
                if target in at:
                    todo.append((at[target], younger))
                if o in ("s_branch", "s_endpgm"):
                    break
                j += 1
    return sorted(bad)


def listing(*ins):
    return [(4 * i, t[0], t[1], 4 * t[2] if len(t) > 2 else None) for i, t in enumerate(ins)]


def test_reads_that_reach_a_barrier_are_found():
    read, bar, end = ("ds_read_b128", " v[0:3], v4"), ("s_barrier", ""), ("s_endpgm", "")
    assert pending_reads(listing(read, bar, end))
    assert not pending_reads(listing(read, ("s_waitcnt", " lgkmcnt(0)"), bar, end))
    assert pending_reads(listing(read, ("s_waitcnt", " vmcnt(0)"), bar, end))
    assert pending_reads(listing(read, read, ("s_waitcnt", " lgkmcnt(1)"), bar, end))
    assert not pending_reads(listing(read, read, ("s_waitcnt", " lgkmcnt(1)"), ("s_waitcnt", " lgkmcnt(0)"), bar, end))
    loop = listing(bar, read, ("s_cbranch_scc1", " 0", 0), ("s_waitcnt", " lgkmcnt(0)"), end)
    assert pending_reads(loop)


@pytest.mark.parametrize("obj", ["vocab_head.o", "topk_logprob.o", "gemm_asm4.o"])
def test_the_built_kernels_have_read_before_every_barrier(check, obj):
    path = os.path.join(CSRC, obj)
    if not os.path.exists(path) or check.objdump() is None:
        pytest.skip("no built objects or no llvm-objdump here")
    kernels = check.functions(path)
    assert sum(any(o == "s_barrier" for _, o, _, _ in code) for code in kernels.values()) >= 3
    for name, code in kernels.items():
        assert not pending_reads(code), name
