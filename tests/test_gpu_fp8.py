"""8-bit block-scaled matrices and their products on the GPU against plain 64-bit forms."""
import numpy as np
import pytest
import torch

import route_case as rc

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def eng():
    import sidekit_amd
    return sidekit_amd.default_engine()


def _wild(shape, dtype, seed):
    t = torch.from_numpy(rc.wild(shape, seed)).to(DT[dtype])
    return t, t.double().numpy()


def _product_close(c, a, b):
    """float32 results: K products, each exact, summed in float32 in any order: K U32 of the sum of magnitudes.
    bf16 and f16 results come from the 8-bit matrix instructions, which add 8 products at a time with the bits below
    2^-13 of the largest of the 8 cut off: of the other 7 less than 7 * 2^-13 of the largest, less than 2^-10 of the 8
    products' magnitudes; added up, 2^-10 of the sum of magnitudes.  That is the worst case; the parts cut off are of
    either sign and no larger than 2^-13 of the products, which bounds the 2-norm of the error by 2^-13 of that of the
    result as long as they do not conspire.  Then the rounding to the result's type (f16: or half its smallest step)."""
    ref = a @ b.T
    mag = np.abs(a) @ np.abs(b).T
    half = rc.half_step(c.dtype)
    d = c.double().cpu().numpy() - ref
    if c.dtype == torch.float32:
        tol = rc.U32 * (a.shape[1] + 1) * mag
    else:
        tol = (2.0 ** -10 + rc.U32 * a.shape[1]) * mag + half * np.abs(ref)
        least = 2.0 ** -25 * np.sqrt(ref.size) if c.dtype == torch.float16 else 0.0
        assert np.linalg.norm(d) <= (half + 2.0 ** -13) * np.linalg.norm(ref) + least
    if c.dtype == torch.float16:
        tol = tol + 2.0 ** -25
    assert (np.abs(d) <= tol).all(), (np.abs(d) - tol).max()


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("M,K", [(1, 1), (3, 127), (17, 128), (5, 129), (130, 640), (33, 1000)])
def test_rows(eng, fmt, dtype, M, K):
    x, x64 = _wild((M, K), dtype, M + K)
    q = eng.fp8_rows(x.cuda(), fmt)
    v, e = rc.fp8_blocks(x64, fmt, 1, 128)
    np.testing.assert_array_equal(q.values().double().cpu().numpy(), v)
    np.testing.assert_array_equal(q.s.cpu().numpy()[:, :e.shape[1]].astype(int) - 127, e)
    assert int(q.q[:, K:].max() if q.q.shape[1] > K else 0) == 0


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("N,K", [(1, 1), (128, 128), (129, 127), (200, 300), (60, 520)])
def test_tiles(eng, fmt, dtype, N, K):
    w, w64 = _wild((N, K), dtype, N + K)
    q, qt = eng.fp8_tiles(w.cuda(), fmt, transposed=True)
    v, e = rc.fp8_blocks(w64, fmt, 128, 128)
    for m, want, es in ((q, v, e), (qt, v.T, e.T)):
        np.testing.assert_array_equal(m.values().double().cpu().numpy(), want)
        np.testing.assert_array_equal(m.s.cpu().numpy()[:, :es.shape[1]].astype(int) - 127, es.repeat(128, 0)[:want.shape[0]])
        assert int(m.q[:, want.shape[1]:].max() if m.q.shape[1] > want.shape[1] else 0) == 0
    only = eng.fp8_tiles(w.cuda(), fmt)
    assert torch.equal(only.q, q.q)


def test_tiles_of_experts(eng):
    w, w64 = _wild((3 * 70, 150), "bf16", 8)
    w, w64 = w.view(3, 70, 150), w64.reshape(3, 70, 150)
    q, qt = eng.fp8_tiles(w.cuda(), transposed=True)
    for e in range(3):
        v, _ = rc.fp8_blocks(w64[e], "e4m3", 128, 128)
        np.testing.assert_array_equal(q.values()[e].double().cpu().numpy(), v)
        np.testing.assert_array_equal(qt.values()[e].double().cpu().numpy(), v.T)


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("R,C", [(1, 1), (128, 128), (127, 200), (300, 61)])
def test_columns(eng, fmt, dtype, R, C):
    x, x64 = _wild((R, C), dtype, R + C)
    q = eng.fp8_columns(x.cuda(), fmt)
    v, _ = rc.fp8_blocks(x64, fmt, 128, 1)
    np.testing.assert_array_equal(q.values().double().cpu().numpy(), v.T)


@pytest.mark.parametrize("T,k,E", [(5, 2, 3), (300, 2, 4), (40, 6, 16), (1, 1, 1)])
@pytest.mark.parametrize("weighted", [False, True])
def test_columns_by_plan(eng, T, k, E, weighted):
    r = np.random.RandomState(T)
    ids = r.randint(-1, E, (T, k)).astype(np.int32)
    if E > 3:
        ids[ids == 2] = 1                                    # an expert without rows
    x, x64 = _wild((T, 70), "bf16", T)
    w = torch.from_numpy(r.rand(T, k)).float()
    plan = eng.route_plan(torch.from_numpy(ids).cuda(), E)
    q = eng.fp8_columns(x.cuda(), plan=plan, weights=w.cuda() if weighted else None)
    got = q.values().double().cpu().numpy()
    pair, expert, _ = rc.plan(ids, E)
    at = 0
    for e in range(E):
        p = pair[expert == e]
        rows = x.float().numpy()[p // k]
        if weighted:
            rows = rows * w.numpy().reshape(-1)[p][:, None]              # a float32 product
        v, _ = rc.fp8_blocks(rows.astype(np.float64), "e4m3", 128, 1)
        np.testing.assert_array_equal(got[:, at:at + p.size], v.T)
        end = at + -(-p.size // 128) * 128
        assert (got[:, at + p.size:end] == 0).all()
        at = end


@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
def test_extreme_blocks(eng, fmt):
    """zeros, the format's borders, float32's ends, infinities and NaN"""
    inf, nan = float("inf"), float("nan")
    x = np.zeros((12, 256), dtype=np.float32)
    x[1, 0], x[1, 130] = rc.TOP[fmt], np.nextafter(np.float32(rc.TOP[fmt]), np.float32(1e9))
    x[2, :] = np.float32(3.4028235e38)
    x[3, :3] = [1e-45, 1e-40, -2e-38]
    x[4, 5], x[4, 6] = inf, 1.0
    x[5, 5], x[5, 6], x[5, 200] = nan, -3.0, -inf
    x[6, :] = np.linspace(-1, 1, 256)
    x[7, :128] = np.exp2(-np.arange(128) / 4.0)
    x[8, :] = 1.0625                                         # ties
    x[9, 0], x[9, 1] = 448, 1e-3
    x[10, 0], x[10, 1] = 1.75, 1.7500001
    x[11, :2] = -0.0
    q = eng.fp8_rows(torch.from_numpy(x).cuda(), fmt)
    v, e = rc.fp8_blocks(x.astype(np.float64), fmt, 1, 128)
    np.testing.assert_array_equal(q.s.cpu().numpy()[:, :2].astype(int) - 127, e)
    # float32's largest number, (2 - 2^-23) 2^127, rounds to 2^128 in four (three) digits: exact in its 8 bits and scale,
    # beyond what float32 values() can show.  Everything else is unchanged by the conversion.
    with np.errstate(over="ignore"):
        v32 = v.astype(np.float32)
    assert (np.isinf(v32) == (np.isinf(v) | (np.abs(v) == 2.0 ** 128))).all() and (v32 == v)[np.isfinite(v32)].all()
    v = v32.astype(np.float64)
    np.testing.assert_array_equal(q.values().double().cpu().numpy(), v)
    qt = eng.fp8_columns(torch.from_numpy(x.T.copy()).cuda(), fmt)
    np.testing.assert_array_equal(qt.values().double().cpu().numpy(), v)


def test_rows_apart(eng):
    big, b64 = _wild((40, 400), "bf16", 3)
    for cols in (slice(8, 264), slice(3, 270)):              # aligned and not
        q = eng.fp8_rows(big.cuda()[:, cols])
        np.testing.assert_array_equal(q.values().double().cpu().numpy(), rc.fp8_blocks(b64[:, cols], "e4m3", 1, 128)[0])
        q = eng.fp8_columns(big.cuda()[:, cols])
        np.testing.assert_array_equal(q.values().double().cpu().numpy(), rc.fp8_blocks(b64[:, cols], "e4m3", 128, 1)[0].T)


SHAPES = [(1, 1, 1), (1, 64, 128), (1, 1000, 4096), (2, 129, 130), (15, 48, 513), (16, 256, 1024), (17, 130, 640), (33, 65, 777),
          (64, 300, 2000), (65, 128, 256), (100, 400, 8000), (127, 127, 127), (128, 128, 128), (129, 257, 385),
          (300, 513, 1152), (512, 512, 512), (700, 260, 2900), (257, 1030, 300)]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_gemm(eng, M, N, K, dtype):
    a, _ = _wild((M, K), "bf16", M + K)
    b, _ = _wild((N, K), "bf16", N + K + 1)
    if dtype == "f16":
        a, b = a / 512, b / 512                              # results inside float16
    A, B = eng.fp8_rows(a.cuda()), eng.fp8_tiles(b.cuda())
    c = eng.gemm_fp8(A, B, dtype=DT[dtype])
    va, vb = A.values().double().cpu().numpy(), B.values().double().cpu().numpy()
    _product_close(c, va, vb)
    assert torch.equal(c, eng.gemm_fp8(a.cuda(), B, dtype=DT[dtype]))        # a float matrix is taken through fp8_rows
    assert torch.equal(c, eng.gemm_fp8(A, B, dtype=DT[dtype]))               # the same bits every time


@pytest.mark.parametrize("M,N,K,dtype", [(4104, 4096, 256, "bf16"),      # a last row tile of 8 rows would begin another round
                                         (4104, 2050, 130, "f32"), (2600, 3100, 384, "bf16"), (2600, 3100, 384, "f32")])
def test_gemm_large_tiles(eng, M, N, K, dtype):
    a, _ = _wild((M, K), "bf16", 11)
    b, _ = _wild((N, K), "bf16", 12)
    A, B = eng.fp8_rows(a.cuda()), eng.fp8_tiles(b.cuda())
    out = torch.full((M + 1, N), 5.0, dtype=DT[dtype]).cuda()
    eng.gemm_fp8(A, B, out=out[:M])
    _product_close(out[:M], A.values().double().cpu().numpy(), B.values().double().cpu().numpy())
    assert (out[M] == 5.0).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_experts_large_tiles(eng, dtype):
    """hundreds of rows an expert: pairs of the plan's tiles, odd numbers of them among the experts"""
    T, k, E, N, K = 3000, 2, 5, 3000, 256
    r = np.random.RandomState(4)
    ids = np.stack([r.choice(E, 2, replace=False, p=[0.35, 0.3, 0.2, 0.1, 0.05]) for _ in range(T)]).astype(np.int32)
    ids[r.rand(T) < 0.1] = -1
    x, _ = _wild((T, K), "bf16", 1)
    w, _ = _wild((E * N, K), "bf16", 2)
    X, W = eng.fp8_rows(x.cuda()), eng.fp8_tiles(w.view(E, N, K).cuda())
    plan = eng.route_plan(torch.from_numpy(ids).cuda(), E)
    rows = eng.gemm_fp8_experts(X, W, plan, dtype=DT[dtype])
    pair, expert, _ = rc.plan(ids, E)
    vx, vw = X.values().double().cpu().numpy(), W.values().double().cpu().numpy()
    for e in range(E):
        m = np.flatnonzero(expert == e)
        _product_close(rows[torch.from_numpy(m).cuda()], vx[pair[m] // k], vw[e])


@pytest.mark.parametrize("fa,fb", [("e4m3", "e5m2"), ("e5m2", "e4m3"), ("e5m2", "e5m2")])
@pytest.mark.parametrize("M,N,K", [(1, 200, 700), (40, 200, 700), (130, 140, 700), (600, 520, 640)])
def test_gemm_formats_and_blocks(eng, fa, fb, M, N, K):
    a, _ = _wild((K, M), "bf16", 1)
    b, _ = _wild((K, N), "f32", 2)
    A, B = eng.fp8_columns(a.cuda(), fa), eng.fp8_columns(b.cuda(), fb)
    c = eng.gemm_fp8(A, B, dtype=torch.float32)
    _product_close(c, A.values().double().cpu().numpy(), B.values().double().cpu().numpy())


@pytest.mark.parametrize("M,N,K", [(1, 64, 4096), (20, 300, 1000), (300, 260, 520), (100, 40, 30720)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_gemm_out_and_accumulate(eng, M, N, K, dtype):
    a, _ = _wild((M, K), "bf16", 5)
    b, _ = _wild((N, K), "bf16", 6)
    A, B = eng.fp8_rows(a.cuda()), eng.fp8_tiles(b.cuda())
    va, vb = A.values().double().cpu().numpy(), B.values().double().cpu().numpy()
    wide = torch.full((M + 2, N + 7), 3.0, dtype=DT[dtype]).cuda()
    out = wide[1:M + 1, 4:N + 4]                             # rows apart, unaligned
    assert eng.gemm_fp8(A, B, out=out).data_ptr() == out.data_ptr()
    _product_close(out, va, vb)
    old = out.double().cpu().numpy()
    eng.gemm_fp8(A, B, out=out, accumulate=True)
    ref = va @ vb.T + old
    mag = np.abs(va) @ np.abs(vb).T + np.abs(old)
    u = rc.U32 * (K + 1) + (2.0 ** -10 if dtype == "bf16" else 0.0)      # as in _product_close
    assert (np.abs(out.double().cpu().numpy() - ref) <= u * mag + rc.half_step(DT[dtype]) * np.abs(ref)).all()
    border = wide.clone()
    border[1:M + 1, 4:N + 4] = 3.0
    assert (border == 3.0).all()                             # nothing beside the result is touched


def test_gemm_nan_stays_in_its_row(eng):
    a, b = torch.randn(40, 256), torch.randn(30, 256)
    a[7, 100] = float("nan")
    a[9, 3] = float("inf")
    c = eng.gemm_fp8(a.cuda(), eng.fp8_tiles(b.cuda()), dtype=torch.float32).cpu()
    bad = torch.zeros(40, dtype=torch.bool)
    bad[[7, 9]] = True
    assert torch.isnan(c[bad]).all() and torch.isfinite(c[~bad]).all()


def test_gemm_empty(eng):
    B = eng.fp8_tiles(torch.randn(30, 256).cuda())
    assert eng.gemm_fp8(torch.empty(0, 256).cuda(), B).shape == (0, 30)


@pytest.mark.parametrize("T,k,E,N,K", [(1, 1, 1, 1, 1), (1, 4, 64, 100, 300), (8, 4, 64, 256, 512), (7, 2, 3, 130, 200), (300, 2, 4, 129, 256),
                                       (500, 3, 5, 64, 640), (64, 6, 8, 200, 130), (1100, 2, 3, 260, 384)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_experts(eng, T, k, E, N, K, dtype):
    r = np.random.RandomState(T + E)
    ids = r.randint(-1, E, (T, k)).astype(np.int32)
    x, _ = _wild((T, K), "bf16", 1)
    w, _ = _wild((E * N, K), "bf16", 2)
    X, W = eng.fp8_rows(x.cuda()), eng.fp8_tiles(w.view(E, N, K).cuda())
    plan = eng.route_plan(torch.from_numpy(ids).cuda(), E)
    rows = eng.gemm_fp8_experts(X, W, plan, dtype=DT[dtype])
    assert torch.equal(rows[:int(plan.offsets[-1])], eng.gemm_fp8_experts(x.cuda(), W, plan, dtype=DT[dtype])[:int(plan.offsets[-1])])
    pair, expert, _ = rc.plan(ids, E)
    vx, vw = X.values().double().cpu().numpy(), W.values().double().cpu().numpy()
    for e in range(E):
        m = expert == e
        if m.any():
            _product_close(rows[torch.from_numpy(np.flatnonzero(m)).cuda()], vx[pair[m] // k], vw[e])
    # rows in the plan's order
    if k > 1 and pair.size:
        xp = torch.zeros(T * k, K, dtype=torch.bfloat16)
        xp[:pair.size] = x[pair // k]
        again = eng.gemm_fp8_experts(xp.cuda(), W, plan, dtype=DT[dtype])
        assert torch.equal(again[:pair.size], rows[:pair.size])


@pytest.mark.parametrize("few", [False, True])
def test_experts_leave_rows_behind_the_last(eng, few):
    """the rows that no pair has keep what the memory held"""
    ids = torch.tensor([[0, -1], [-1, -1], [1, 0]], dtype=torch.int32)
    plan = eng.route_plan(ids.cuda(), 2)
    assert plan.more_rows == 16
    W = eng.fp8_tiles(torch.randn(2, 40, 128).cuda())
    X = eng.fp8_rows(torch.randn(3, 128).cuda())
    out = torch.full((6, 40), 7.0).cuda()
    eng._check(eng.lib.skm_gemm_fp8_experts(
        eng.ctx, X.q.data_ptr(), X.s.data_ptr(), 0, -1, 0, 3, W.q.data_ptr(), W.s.data_ptr(), 0, 2, 40, 128,
        plan._ptr("pair"), 2, 6, plan._ptr("first"), plan._ptr("tiles"), 16 if few else 0, plan._ptr("more_tiles"),
        plan._ptr("more_count"), out.data_ptr(), 0, None, 0, eng._stream()))
    assert (out[3:] == 7.0).all() and not (out[:3] == 7.0).any()


@pytest.mark.parametrize("T,k,E,N,K", [(1, 1, 1, 1, 1), (5, 2, 9, 40, 70), (300, 2, 4, 129, 200), (900, 3, 3, 64, 300)])
def test_experts_wgrad(eng, T, k, E, N, K):
    r = np.random.RandomState(T)
    ids = r.randint(-1, E, (T, k)).astype(np.int32)
    x, _ = _wild((T, K), "bf16", 1)
    dy, _ = _wild((T, N), "bf16", 2)
    w = torch.from_numpy(r.rand(T, k)).float()
    plan = eng.route_plan(torch.from_numpy(ids).cuda(), E)
    A = eng.fp8_columns(dy.cuda(), "e5m2", plan=plan, weights=w.cuda())
    B = eng.fp8_columns(x.cuda(), plan=plan)
    dw = eng.gemm_fp8_experts_wgrad(A, B, plan)
    va, vb = A.values().double().cpu().numpy(), B.values().double().cpu().numpy()
    first = plan.first.cpu().numpy()
    for e in range(E):
        sl = slice(first[e] * 128, first[e + 1] * 128)
        if sl.start == sl.stop:
            assert (dw[e] == 0).all()
        else:
            _product_close(dw[e], va[:, sl], vb[:, sl])
    old = dw.clone()
    eng.gemm_fp8_experts_wgrad(A, B, plan, out=dw, accumulate=True)
    assert torch.equal(dw, 2 * old)                          # the same sums, added to themselves
