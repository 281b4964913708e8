"""Routing (route, route_backward, route_plan, route_combine) on the GPU against plain 64-bit forms."""
import numpy as np
import pytest
import torch

import route_case as rc

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "f64": torch.float64}


@pytest.fixture(scope="module")
def eng():
    import sidekit_amd
    return sidekit_amd.default_engine()


def _logits(T, E, dtype, seed, masked, spread=2.0):
    r = np.random.RandomState(seed)
    x = r.randn(T, E) * spread
    if masked:
        x[r.rand(T, E) < 0.2] = -np.inf
        x[r.rand(T) < 0.2] = -np.inf
        if T > 2:
            x[0] = -np.inf
            x[1, 1:] = -np.inf                      # one expert left
    t = torch.from_numpy(x).to(DT[dtype])
    return t, t.double().numpy()


def _check_weights(w, rw, x, ids, scale):
    """w = scale t / sum t (or p): exp of a float32 difference d has a relative error of U32 (|d| + a few), the sum of
    positive terms no more than its terms, and there are two divisions / products and one rounding: U32 (2 |d| + 16)."""
    xs = np.take_along_axis(x, np.where(ids >= 0, ids, 0), 1)
    xs = np.where(ids >= 0, xs, 0.0)
    top = np.where(np.isfinite(x), x, -1e9).max(1, keepdims=True)
    d = np.minimum(np.abs(xs - np.where(top < -1e8, 0.0, top)) + np.abs(xs), 200.0)
    tol = rc.U32 * (2 * d + 16) * np.abs(rw) + 1e-37
    assert (np.abs(w - rw) <= tol).all(), np.abs(w - rw).max()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16", "f64"])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 64, 4), (3, 7, 7), (5, 65, 3), (130, 128, 8), (67, 256, 8), (33, 513, 20),
                                   (9, 2049, 33), (5, 4096, 64), (257, 16, 1)])
@pytest.mark.parametrize("scores,bias,renorm,masked", [("softmax", False, True, False), ("softmax", True, False, True),
                                                       ("sigmoid", True, True, True), ("sigmoid", False, False, False)])
def test_route(eng, dtype, T, E, k, scores, bias, renorm, masked):
    x, x64 = _logits(T, E, dtype, T * 1000 + E, masked)
    b = torch.from_numpy(np.random.RandomState(5).randn(E) * 0.1).float() if bias else None
    ids, w = eng.route(x.cuda(), k, scores=scores, bias=b.cuda() if bias else None, renorm=renorm, scale=1.5)
    rids, rw, _ = rc.route(x64, k, scores, b.numpy() if bias else None, renorm=renorm, scale=1.5)
    np.testing.assert_array_equal(ids.cpu().numpy(), rids)
    _check_weights(w.cpu().numpy().astype(np.float64), rw, x64, rids, 1.5)


@pytest.mark.parametrize("E,groups,group_k,k,top", [(64, 8, 4, 6, 2), (256, 8, 3, 8, 2), (24, 4, 1, 5, 1), (60, 20, 7, 9, 2),
                                                    (8, 8, 3, 3, 2), (384, 8, 8, 10, 2), (128, 64, 5, 4, 1)])
@pytest.mark.parametrize("scores,bias,masked", [("softmax", False, True), ("sigmoid", True, False), ("sigmoid", True, True),
                                                ("softmax", True, False)])
def test_route_groups(eng, E, groups, group_k, k, top, scores, bias, masked):
    x, x64 = _logits(201, E, "f32", E + groups, masked)
    b = torch.from_numpy(np.random.RandomState(6).randn(E) * 0.2).float() if bias else None
    ids, w = eng.route(x.cuda(), k, scores=scores, bias=b.cuda() if bias else None, groups=groups, group_k=group_k,
                       group_top=top)
    rids, rw, _ = rc.route(x64, k, scores, b.numpy() if bias else None, groups, group_k, top)
    np.testing.assert_array_equal(ids.cpu().numpy(), rids)
    _check_weights(w.cpu().numpy().astype(np.float64), rw, x64, rids, 1.0)


def test_route_ties_and_near_ties(eng):
    """Equal choices go to the lowest index; choices that a float32 evaluation cannot tell apart keep their order."""
    T, E, k = 64, 96, 9
    r = np.random.RandomState(3)
    x = np.round(r.randn(T, E) * 2) / 2                                  # many equal logits
    ids, _ = eng.route(torch.from_numpy(x).float().cuda(), k)
    np.testing.assert_array_equal(ids.cpu().numpy(), rc.route(x, k)[0])
    # p + bias equal but for 1e-9: the bias of expert e is what is missing to a common value
    x = r.randn(1, E).astype(np.float32).astype(np.float64)
    p = 1 / (1 + np.exp(-x[0]))
    b = (2.0 - p).astype(np.float32)                                     # c = 2 up to the rounding of b: 1e-7 apart
    xs = np.repeat(x, T, 0)
    ids, _ = eng.route(torch.from_numpy(xs).float().cuda(), k, scores="sigmoid", bias=torch.from_numpy(b).cuda())
    np.testing.assert_array_equal(ids.cpu().numpy(), rc.route(xs, k, "sigmoid", b)[0])
    # float64 logits that agree in float32
    x = 5.0 + r.permutation(T * E).reshape(T, E) * 1e-12
    ids, _ = eng.route(torch.from_numpy(x).cuda(), k)
    np.testing.assert_array_equal(ids.cpu().numpy(), rc.route(x, k)[0])
    # zeros of either sign are one number; whole rows of equal logits
    for dt in (torch.bfloat16, torch.float32, torch.float64):
        z = torch.zeros(T, E, dtype=dt)
        z[r.rand(T, E) < 0.5] = -0.0
        z[3] = 1.5
        ids, w = eng.route(z.cuda(), k)
        assert ids.cpu().tolist() == [list(range(k))] * T
        assert (torch.abs(w.cpu().double() - 1 / k) <= 4 * rc.U32 / k).all()
    # groups whose scores differ by 1e-9
    x = np.tile(r.randn(T, 12), (1, 8)) + r.randn(T, 96) * 1e-9
    b = (r.randn(96) * 0.1).astype(np.float32)
    b = np.tile(b[:12], 8)
    ids, _ = eng.route(torch.from_numpy(x).cuda(), k, bias=torch.from_numpy(b).cuda(), groups=8, group_k=3)
    np.testing.assert_array_equal(ids.cpu().numpy(), rc.route(x, k, "softmax", b, 8, 3)[0])


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_route_many_rows(eng, scores):
    """more rows than a launch has workgroups at once, the last workgroup partly filled; float32 and half-precision"""
    for dtype, T, E, k, bias, groups, group_k in (("f32", 20011, 256, 8, True, 8, 4), ("bf16", 30001, 128, 8, True, 1, 1),
                                                  ("f64", 5003, 512, 20, False, 1, 1), ("f16", 4099, 300, 3, True, 6, 2)):
        x, x64 = _logits(T, E, dtype, T, False, 1.5)
        b = (np.random.RandomState(8).randn(E) * 0.05).astype(np.float32) if bias else None
        ids, w = eng.route(x.cuda(), k, scores=scores, bias=torch.from_numpy(b).cuda() if bias else None, groups=groups,
                           group_k=group_k)
        rids, rw, _ = rc.route(x64, k, scores, b, groups, group_k)
        np.testing.assert_array_equal(ids.cpu().numpy(), rids)
        _check_weights(w.cpu().numpy().astype(np.float64), rw, x64, rids, 1.0)


@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_route_special_values(eng, scores):
    inf, nan = float("inf"), float("nan")
    x = np.zeros((8, 6))
    x[0, 2] = nan
    x[1, 3] = inf
    x[2] = -inf
    x[3, 1:] = -inf
    x[4] = [-300, -301, -299.5, -310, -500, -400]           # far below what float32 exponentials reach
    x[5] = [80, 81, 79, 3, -88, -104]
    x[6] = 3.4e38
    x[7] = [-3e38, 3e38, 0, 1, -1, 2]
    t = torch.from_numpy(x).float()
    for renorm in (True, False):
        ids, w = eng.route(t.cuda(), 4, scores=scores, renorm=renorm)
        rids, rw, _ = rc.route(t.double().numpy(), 4, scores, renorm=renorm)
        w = w.cpu().numpy().astype(np.float64)
        np.testing.assert_array_equal(ids.cpu().numpy(), rids)
        np.testing.assert_array_equal(np.isnan(w), np.isnan(rw))
        ok = ~np.isnan(rw)
        assert (np.abs(w - rw)[ok] <= rc.U32 * 900 * np.abs(rw)[ok] + 1e-37).all()
    # an expert whose bias is -inf is never chosen
    b = torch.zeros(6)
    b[0] = -inf
    ids, _ = eng.route(torch.zeros(3, 6).cuda(), 6, scores=scores, bias=b.cuda())
    assert ids.cpu().tolist() == [[1, 2, 3, 4, 5, -1]] * 3


def test_route_rows_apart_and_empty(eng):
    big = torch.randn(50, 300, generator=torch.Generator().manual_seed(1))
    x = big.cuda()[:, 3:70]                                  # rows 300 apart, not aligned
    ids, w = eng.route(x, 5)
    rids, rw, _ = rc.route(big[:, 3:70].double().numpy(), 5)
    np.testing.assert_array_equal(ids.cpu().numpy(), rids)
    dx = eng.route_backward(x, ids, torch.ones_like(w), renorm=False)
    ref, mag = rc.route_backward(big[:, 3:70].double().numpy(), rids, np.ones((50, 5)), renorm=False)
    assert (np.abs(dx.cpu().numpy() - ref) <= rc.U32 * 64 * mag).all()
    ids, w = eng.route(torch.empty(0, 8).cuda(), 2)
    assert ids.shape == (0, 2) and w.shape == (0, 2)
    assert eng.route_backward(torch.empty(0, 8).cuda(), ids, w).shape == (0, 8)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16", "f64"])
@pytest.mark.parametrize("T,E,k", [(1, 8, 2), (70, 64, 6), (33, 257, 8), (5, 1100, 20), (3, 4096, 64)])
@pytest.mark.parametrize("scores,renorm", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
def test_route_backward(eng, dtype, T, E, k, scores, renorm):
    x, x64 = _logits(T, E, dtype, T + E, T > 2)
    ids = rc.route(x64, k, scores)[0]
    r = np.random.RandomState(9)
    if T > 2:
        ids[1, 0], ids[2, 0] = E + 3, -7                     # outside: empty places
        if k > 1:
            ids[T - 1, 0] = ids[T - 1, 1]                    # the same expert twice
    g = r.randn(T, k).astype(np.float32)
    dx = eng.route_backward(x.cuda(), torch.from_numpy(ids).cuda(), torch.from_numpy(g).cuda(), scores=scores,
                            renorm=renorm, scale=2.5)
    assert dx.dtype == DT[dtype]
    ref, mag = rc.route_backward(x64, ids, g, scores, renorm, 2.5)
    u = 2.0 ** -53 if dtype == "f64" else rc.U32
    # exponentials of differences up to |d| ~ 12 (U (|d| + 4) each, numerator and sum), sums of E and k terms in trees,
    # five more products: under 64 U of the magnitudes; then the rounding to the gradient's type
    tol = u * (64 + E / 32) * mag + rc.half_step(DT[dtype]) * np.abs(ref) + (3e-8 if dtype == "f16" else 1e-37)
    assert (np.abs(dx.double().cpu().numpy() - ref) <= tol).all()


def test_route_backward_against_differences(eng):
    x, x64 = _logits(6, 20, "f64", 4, False)
    g = np.random.RandomState(2).randn(6, 5).astype(np.float32)
    for scores in ("softmax", "sigmoid"):
        for renorm in (True, False):
            ids, w = eng.route(x.cuda(), 5, scores=scores, renorm=renorm)
            dx = eng.route_backward(x.cuda(), ids, torch.from_numpy(g).cuda(), scores=scores, renorm=renorm).cpu().numpy()
            h = 1e-5
            for e in range(20):
                a, b = x64.copy(), x64.copy()
                a[:, e] += h
                b[:, e] -= h
                ra, rb = rc.route(a, 5, scores, renorm=renorm), rc.route(b, 5, scores, renorm=renorm)
                assert (ra[0] == ids.cpu().numpy()).all() and (rb[0] == ra[0]).all()
                num = ((ra[1] - rb[1]) * g).sum(1) / (2 * h)
                # h^2 / 6 of a third derivative below 10 |g|, and 2^-53 / h
                assert (np.abs(num - dx[:, e]) <= 1e-8).all()


@pytest.mark.parametrize("T,k,E", [(1, 1, 1), (1, 4, 64), (0, 2, 5), (9, 3, 5), (700, 6, 64), (1025, 4, 4), (3000, 8, 130),
                                   (40000, 2, 16), (30001, 2, 512), (20000, 3, 600), (65536, 1, 3), (65537, 1, 3),
                                   (5000, 3, 4096), (300, 2, 2500), (70001, 8, 257)])
def test_plan(eng, T, k, E):
    r = np.random.RandomState(T + E)
    ids = r.randint(-1, E, (T, k)).astype(np.int32)
    if T > 8:
        ids[3] = E                                           # outside
        ids[r.rand(T) < 0.3] = E // 2                        # one popular expert, also twice in a row
    plan = eng.route_plan(torch.from_numpy(ids).cuda(), E)
    pair, expert, pos = rc.plan(ids, E)
    n = pair.size
    np.testing.assert_array_equal(plan.pair.cpu().numpy()[:n], pair)
    np.testing.assert_array_equal(plan.pos.cpu().numpy(), pos)
    count = np.bincount(expert, minlength=E)
    np.testing.assert_array_equal(plan.offsets.cpu().numpy(), np.concatenate([[0], count.cumsum()]))
    for rows, name in ((128, "tiles"), (plan.more_rows, "more_tiles")):
        if rows == 0:
            continue
        nt = -(-count // rows)
        if name == "tiles":
            np.testing.assert_array_equal(plan.first.cpu().numpy(), np.concatenate([[0], nt.cumsum()]))
        else:
            assert int(plan._view("more_count")[0]) == nt.sum()
        want = [(e, count[:e].sum() + i * rows, min(rows, count[e] - i * rows), 0) for e in range(E) for i in range(nt[e])]
        got = plan._view(name).view(-1, 4).cpu().numpy()[:len(want)]
        np.testing.assert_array_equal(got, np.array(want, dtype=np.int64).reshape(-1, 4))
        assert len(want) <= plan._view(name).numel() // 4


@pytest.mark.parametrize("rows_dt,out_dt", [("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"),
                                            ("bf16", "f32"), ("f16", "f16"), ("f16", "f32")])
@pytest.mark.parametrize("T,k,E,N", [(1, 1, 1, 1), (5, 3, 4, 37), (130, 4, 8, 256), (33, 8, 16, 1000)])
def test_combine(eng, rows_dt, out_dt, T, k, E, N):
    r = np.random.RandomState(T + N)
    ids = r.randint(-1, E, (T, k)).astype(np.int32)
    plan = eng.route_plan(torch.from_numpy(ids).cuda(), E)
    rows = torch.from_numpy(r.randn(T * k, N)).to(DT[rows_dt])
    pair, _, pos = rc.plan(ids, E)
    rows[pair.size:] = float("nan")                          # what is behind the rows is not looked at
    w = torch.from_numpy(r.randn(T, k)).float()
    out = eng.route_combine(rows.cuda(), w.cuda(), plan, dtype=DT[out_dt])
    terms = np.where((pos >= 0)[:, :, None], rows.double().numpy()[np.where(pos >= 0, pos, 0)], 0.0) * w.double().numpy()[:, :, None]
    tol = rc.U32 * (k + 1) * np.abs(terms).sum(1) + rc.half_step(DT[out_dt]) * np.abs(terms.sum(1)) + 1e-7 * (out_dt == "f16")
    assert (np.abs(out.double().cpu().numpy() - terms.sum(1)) <= tol).all()
    dout = torch.from_numpy(r.randn(T, N)).to(DT[out_dt])
    dw = eng.route_combine_backward(rows.cuda(), dout.cuda(), plan).double().cpu().numpy()
    terms = np.where((pos >= 0)[:, :, None], rows.double().numpy()[np.where(pos >= 0, pos, 0)], 0.0) * dout.double().numpy()[:, None, :]
    assert (np.abs(dw - terms.sum(2)) <= rc.U32 * (N + 1) * np.abs(terms).sum(2)).all()


def test_combine_keeps_nan_of_a_row_without_choice(eng):
    x = torch.zeros(3, 8)
    x[1, 4] = float("nan")
    ids, w = eng.route(x.cuda(), 2)
    plan = eng.route_plan(ids, 8)
    out = eng.route_combine(torch.ones(6, 5).cuda(), w, plan)
    assert torch.isnan(out[1]).all() and torch.isfinite(out[[0, 2]]).all()


def test_combine_refuses_mixed_halves(eng):
    import sidekit_amd
    plan = eng.route_plan(torch.zeros(2, 1, dtype=torch.int32).cuda(), 1)
    with pytest.raises(sidekit_amd.SkmError):
        eng.route_combine(torch.zeros(2, 4, dtype=torch.bfloat16).cuda(), torch.zeros(2, 1).cuda(), plan, dtype=torch.float16)
    with pytest.raises(sidekit_amd.SkmError):
        eng.route(torch.zeros(2, 4), 1)                      # a host tensor
