"""Up to 512 experts, 16 lanes a row, groups whose scores float32 cannot tell apart: which are the best is decided in float64,
for every number of groups that a row's lanes hold."""
import numpy as np
import pytest
import torch

import route_case as rc
from test_gpu_route import DT, _check_weights

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    import sidekit_amd
    return sidekit_amd.default_engine()


def _apart(c, groups, top):
    """rows in which any two groups' scores are sums of the very same numbers (a tie in any arithmetic) or further apart than
    the last bits of a float64 exponential and sum"""
    T, E = c.shape
    best = np.sort(c.reshape(T, groups, E // groups), 2)[:, :, -top:]
    score = best.sum(2)
    order = np.argsort(score, 1)
    gap = np.diff(np.take_along_axis(score, order, 1), axis=1)
    same = (np.diff(np.take_along_axis(best, order[:, :, None], 1), axis=1) == 0).all(2)
    return (same | (gap > 1e-12 * np.abs(score).max(1, keepdims=True))).all(1)


@pytest.mark.parametrize("groups,group_k", [(2, 1), (3, 2), (4, 1), (4, 3), (5, 2), (8, 3), (8, 7), (12, 5), (15, 4), (16, 9)])
@pytest.mark.parametrize("per,k,top", [(1, 1, 2), (5, 3, 1), (16, 4, 2), (32, 8, 2)])
@pytest.mark.parametrize("dtype,scores,bias", [("f32", "softmax", False), ("f32", "sigmoid", False), ("f32", "softmax", True),
                                               ("bf16", "sigmoid", True), ("f16", "softmax", True)])
def test_near_groups(eng, groups, group_k, per, k, top, dtype, scores, bias):
    T, E = 60, groups * per
    r = np.random.RandomState(E + group_k)
    x = np.tile(r.randn(T, 1, per) * 2, (1, groups, 1))
    if not bias:
        x += r.randint(-3, 4, x.shape) * 2.0 ** -21         # bits that a float32 of this size holds
    t = torch.from_numpy(x.reshape(T, E)).to(DT[dtype])
    x = t.double().numpy()
    # with a bias: what differs between the groups is the bias, by up to 2^-22
    b = (r.rand(E) * 2.0 ** -22).astype(np.float32) if bias else None
    e = np.exp(x - x.max(1, keepdims=True))
    p = e / e.sum(1, keepdims=True) if scores == "softmax" else 1 / (1 + np.exp(-x))
    keep = _apart(p + b.astype(np.float64) if bias else p, groups, top)
    assert keep.sum() >= T // 2
    x, t = x[keep], t[torch.from_numpy(keep)]
    ids, w = eng.route(t.cuda(), min(k, per * group_k), scores=scores, bias=torch.from_numpy(b).cuda() if bias else None,
                       groups=groups, group_k=group_k, group_top=top)
    rids, rw, _ = rc.route(x, min(k, per * group_k), scores, b, groups, group_k, top)
    np.testing.assert_array_equal(ids.cpu().numpy(), rids)
    _check_weights(w.cpu().numpy().astype(np.float64), rw, x, rids, 1.0)


@pytest.mark.parametrize("groups,group_k", [(2, 1), (4, 2), (8, 2), (8, 5), (16, 3)])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_saturated_groups(eng, groups, group_k, dtype):
    """sigmoids that float32 rounds to 1 and float64 does not"""
    T, per = 300, 4
    r = np.random.RandomState(groups)
    x = np.round(r.uniform(17, 24, (T, groups * per)) * 8) / 8
    keep = _apart(1 / (1 + np.exp(-x)), groups, 2)
    x = x[keep]
    assert keep.sum() >= T // 2
    ids, _ = eng.route(torch.from_numpy(x).to(DT[dtype]).cuda(), 4, scores="sigmoid", groups=groups, group_k=group_k)
    np.testing.assert_array_equal(ids.cpu().numpy(), rc.route(x, 4, "sigmoid", None, groups, group_k)[0])
