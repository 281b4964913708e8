"""tools/isa_lint.py, rule iii: a kernel may hold loops over LDS rings of different depth; each is held to its own."""
import os
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "tools"))
import isa_lint  # noqa: E402

NAME = "_Z10k_gemm_fp8ILi4ELi2ELi0ELi0EfEv7Fp8Args"


def _loop(wait):
    """load into the ring, wait, barrier, read, around again (two words each way)"""
    lines = [("s_nop", "0"), ("global_load_lds_dwordx4", "v[2:3], off"), ("s_waitcnt", wait), ("s_barrier", ""),
             ("ds_read_b128", "v[4:7], v1"), ("s_cbranch_scc1", "%d" % (0x10000 - 5)), ("s_endpgm", "")]
    return [isa_lint.Ins(op, args, 0x1000 + 4 * k) for k, (op, args) in enumerate(lines)]


def test_three_stages_by_the_loop():
    # the three-stage loop of the 256 x 128 kernel waits until 14 loads are left; here 14 would never be exceeded, so the
    # reads two iterations on are not covered, those three on are the ones that count
    deep = isa_lint.ring_depth(NAME, _loop("vmcnt(14)"))
    # the loop of its half tile has two stages and waits for everything
    flat = isa_lint.ring_depth(NAME, _loop("vmcnt(0)"))
    assert (deep, flat) == (3, 2)
    assert isa_lint.ring_depth("_Z10k_gemm_fp8ILi4ELi4ELi0ELi0EDF16bEv7Fp8Args", _loop("vmcnt(14)")) == 2
    assert isa_lint.ring_depth("k_gemm_b3", _loop("vmcnt(6)")) == 2
    assert isa_lint.ring_depth("k_estep_fat", _loop("vmcnt(0)")) == 1


def test_two_stage_loop_of_a_three_stage_kernel():
    """a two-stage loop that leaves one load in flight too many: reachable two iterations on, unseen at a depth of three"""
    lines = [("s_nop", "0")]
    for _ in range(2):          # two iterations' loads in flight at the wait, where one must have arrived
        lines += [("global_load_lds_dwordx4", "v[2:3], off")]
    lines += [("s_waitcnt", "vmcnt(5)"), ("s_barrier", ""), ("ds_read_b128", "v[4:7], v1"),
              ("s_cbranch_scc1", "%d" % (0x10000 - 6)), ("s_endpgm", "")]
    ins = [isa_lint.Ins(op, args, 0x1000 + 4 * k) for k, (op, args) in enumerate(lines)]
    assert any(f.startswith("(iii)") for f in isa_lint.lint_kernel(NAME, ins))
    # two loads an iteration: those of the one before are covered
    good = [isa_lint.Ins(a.op, "vmcnt(2)" if a.op == "s_waitcnt" else a.args, a.addr) for a in ins]
    assert isa_lint.lint_kernel(NAME, good) == []
