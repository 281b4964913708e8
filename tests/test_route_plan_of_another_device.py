"""A plan is tables in one device's memory: a call on another device, or with something that is no plan, is refused before
the tables are handed to a kernel."""
import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
import sidekit_amd as sk        # noqa: E402


class _Engine(sk.HipEngine):
    def __init__(self, device):
        self.torch, self.lib, self.device = torch, sk.load_library(), torch.device(device)
        self.ctx = None                              # the library refuses a call without a context
        self._dt_codes = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2, torch.float64: 3}

    def _raw_stream(self):
        return None

    def close(self):
        pass


@pytest.mark.parametrize("wrong", ["device", "kind"])
def test_plan(wrong):
    eng = _Engine("cpu")
    good = sk.RoutePlan(eng, 4, 2, 3)
    plan = sk.RoutePlan(_Engine("meta"), 4, 2, 3) if wrong == "device" else {"T": 4}
    x, rows, g = torch.zeros(4, 8), torch.zeros(8, 6), torch.zeros(4, 2)
    W = sk.Fp8Matrix(eng, (3, 6), 8, "e4m3")
    columns = sk.Fp8Matrix(eng, (6,), good.max_tiles * 128, "e4m3")
    columns.plan = plan
    for call in (lambda p: eng.route_combine(rows, g, p), lambda p: eng.route_combine_backward(rows, torch.zeros(4, 6), p),
                 lambda p: eng.fp8_columns(x, plan=p), lambda p: eng.gemm_fp8_experts(x, W, p),
                 lambda p: eng.gemm_fp8_experts_wgrad(columns, columns, p)):
        with pytest.raises(sk.SkmError, match="RoutePlan"):
            call(plan)
    # the right one reaches the library, which wants a context
    with pytest.raises(sk.SkmError, match="bad argument"):
        eng.route_combine(rows, g, good)
