"""Sizes and options beyond the 32-bit integers of the C entry points are refused by the engine's methods (ctypes would cut
them to their low bits, and the call would work on a part of its operands), on an engine of tensors without memory."""
import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
import sidekit_amd as sk        # noqa: E402

BIG = 2 ** 32 + 8               # 8 in the low 32 bits


class _MetaEngine(sk.HipEngine):
    def __init__(self):
        self.torch, self.lib, self.device = torch, sk.load_library(), torch.device("meta")
        self.ctx = None                              # the library refuses a call without a context
        self._dt_codes = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2, torch.float64: 3}

    def _raw_stream(self):
        return None

    def close(self):
        pass


@pytest.fixture(scope="module")
def eng():
    return _MetaEngine()


def _matrix(rows, cols, dtype=torch.float32):
    return torch.empty(rows, cols, dtype=dtype, device="meta")


def _refused(f, *a, **kw):
    with pytest.raises(sk.SkmError, match=r"2\^31"):
        f(*a, **kw)


def test_columns(eng):
    x = _matrix(2, BIG)
    ids, g = _matrix(2, 2, torch.int32), _matrix(2, 2)
    _refused(eng.route, x, 2)
    _refused(eng.route_backward, x, ids, g)
    _refused(eng.route_backward, _matrix(2, 8), _matrix(2, BIG, torch.int32), _matrix(2, BIG))
    _refused(eng.fp8_rows, x)
    _refused(eng.fp8_columns, x)
    plan = sk.RoutePlan(eng, 2, 1, 3)
    _refused(eng.route_combine, x, _matrix(2, 1), plan)
    _refused(eng.route_combine_backward, x, x, plan)


def test_rows_and_matrices(eng):
    _refused(eng.fp8_tiles, _matrix(BIG, 8))
    _refused(eng.fp8_tiles, _matrix(8, BIG))
    _refused(eng.fp8_tiles, torch.empty(BIG, 1, 1, device="meta"))
    B = sk.Fp8Matrix(eng, (6,), 8, "e4m3")
    _refused(eng.gemm_fp8, _matrix(BIG, 8), B)
    _refused(eng.gemm_fp8, sk.Fp8Matrix(eng, (BIG,), 8, "e4m3"), B)
    _refused(eng.gemm_fp8, _matrix(8, 8), sk.Fp8Matrix(eng, (BIG,), 8, "e4m3"))


@pytest.mark.parametrize("kw", [dict(k=BIG), dict(k=2 - 2 ** 32), dict(groups=2 ** 32 + 1), dict(groups=4, group_k=2 ** 32 + 2),
                                dict(group_top=2 ** 32 + 1), dict(group_top=1 - 2 ** 32)])
def test_options(eng, kw):
    a = dict(k=2)
    a.update(kw)
    _refused(eng.route, _matrix(4, 8), **a)


def test_experts(eng):
    _refused(eng.route_plan, _matrix(4, 2, torch.int32), BIG)
    _refused(eng.route_plan, _matrix(4, BIG, torch.int32), 8)


def test_smaller_ones_reach_the_library(eng):
    for f in (lambda: eng.route(_matrix(4, 8), 2), lambda: eng.fp8_rows(_matrix(4, 8)),
              lambda: eng.gemm_fp8(_matrix(4, 8), sk.Fp8Matrix(eng, (6,), 8, "e4m3"))):
        with pytest.raises(sk.SkmError, match="bad argument"):
            f()
