"""Groups of more than 512 experts (a wave a row), of float64 logits (float64 throughout) and of half-precision logits; groups
whose scores float32 cannot tell apart."""
import numpy as np
import pytest
import torch

import route_case as rc
from test_gpu_route import DT, _check_weights, _logits

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    import sidekit_amd
    return sidekit_amd.default_engine()


@pytest.mark.parametrize("E,groups,group_k,k,top", [(1024, 16, 5, 8, 2), (1000, 8, 3, 20, 2), (2048, 64, 7, 8, 2), (4096, 32, 4, 9, 1),
                                                    (520, 40, 11, 13, 2), (256, 8, 3, 8, 2), (24, 4, 2, 6, 1)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16", "f64"])
@pytest.mark.parametrize("scores,bias,masked", [("softmax", False, True), ("softmax", True, False), ("sigmoid", True, True),
                                                ("sigmoid", False, False)])
def test_groups(eng, E, groups, group_k, k, top, dtype, scores, bias, masked):
    x, x64 = _logits(41, E, dtype, E + groups, masked)
    b = torch.from_numpy(np.random.RandomState(6).randn(E) * 0.2).float() if bias else None
    ids, w = eng.route(x.cuda(), k, scores=scores, bias=b.cuda() if bias else None, groups=groups, group_k=group_k,
                       group_top=top, scale=1.5)
    rids, rw, _ = rc.route(x64, k, scores, b.numpy() if bias else None, groups, group_k, top, scale=1.5)
    np.testing.assert_array_equal(ids.cpu().numpy(), rids)
    _check_weights(w.cpu().numpy().astype(np.float64), rw, x64, rids, 1.5)


@pytest.mark.parametrize("E,groups,group_k,k", [(1024, 16, 5, 8), (2048, 64, 20, 8), (768, 8, 3, 4), (1000, 8, 4, 20)])
@pytest.mark.parametrize("dtype", ["f32", "f64"])
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_near_groups(eng, E, groups, group_k, k, dtype, scores):
    """Every group holds the same logits but for a few last bits, so that the groups' scores differ by less than float32
    arithmetic resolves; which are the best is decided in float64.  The oracle's float64 sums of the softmax are good to
    2^-53 E; scores are kept further apart than that by the rows that are taken."""
    T, per = 40, E // groups
    r = np.random.RandomState(E + groups)
    x = np.tile(r.randn(T, 1, per) * 2, (1, groups, 1))
    x += r.randint(-3, 4, x.shape) * 2.0 ** -21            # bits that a float32 of this size holds
    x = x.reshape(T, E).astype(np.float32).astype(np.float64)
    p = np.exp(x - x.max(1, keepdims=True))
    p = p / p.sum(1, keepdims=True) if scores == "softmax" else 1 / (1 + np.exp(-x))
    score = np.sort(p.reshape(T, groups, per), 2)[:, :, -2:].sum(2)
    gap = np.diff(np.sort(score, 1), axis=1)
    # equal pairs of the two largest logits are a tie, which goes to the lower group; otherwise the gap counts
    apart = ((gap == 0) | (gap > 1e-12 * score.max(1, keepdims=True))).all(1)
    assert apart.sum() > T // 2
    x = x[apart]
    ids, w = eng.route(torch.from_numpy(x).to(DT[dtype]).cuda(), k, scores=scores, groups=groups, group_k=group_k)
    rids, rw, _ = rc.route(x, k, scores, None, groups, group_k)
    same = (ids.cpu().numpy() == rids).all(1)
    # a row of tied groups: their scores are sums of the same two numbers, in the oracle's order of addition the same too
    np.testing.assert_array_equal(same, np.ones(len(same), dtype=bool))
    _check_weights(w.cpu().numpy().astype(np.float64), rw, x, rids, 1.0)
