"""A plan of no pairs, for every way in which a plan of its number of experts is made."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    import sidekit_amd
    return sidekit_amd.default_engine()


@pytest.mark.parametrize("k,E", [(1, 1), (2, 2048), (2, 2049), (2, 2500), (1, 4096)])
def test_no_pairs(eng, k, E):
    plan = eng.route_plan(torch.empty(0, k, dtype=torch.int32, device="cuda"), E)
    for name in ("offsets", "first", "more_count"):
        assert (plan._view(name) == 0).all()
    assert plan.pos.shape == (0, k) and plan.pair.numel() == 0 and plan.tiles.shape[0] == 0


def test_chain_without_tokens_over_many_experts(eng):
    E, N, K = 2500, 6, 10
    ids, w = eng.route(torch.empty(0, E, device="cuda"), 2)
    plan = eng.route_plan(ids, E)
    W = eng.fp8_tiles(torch.ones(E, N, K, device="cuda"))
    x = torch.empty(0, K, device="cuda")
    rows = eng.gemm_fp8_experts(x, W, plan)
    assert eng.route_combine(rows, w, plan).shape == (0, N)
    dy = torch.empty(0, N, device="cuda")
    dw = eng.gemm_fp8_experts_wgrad(eng.fp8_columns(dy, plan=plan), eng.fp8_columns(x, plan=plan), plan)
    assert dw.shape == (E, N, K) and (dw == 0).all()
