"""Every kernel of the 8-bit products on sums that are long enough for its ring of LDS stages to go round and its scale groups
(four blocks) to change, with last row tiles on both sides of half a tile, either 8-bit format and each result type.  The
sizes are those that the rules on a GPU of 256 compute units send to the kernel named beside them; elsewhere they are ordinary
products.  References and tolerances as in test_gpu_fp8."""
import numpy as np
import pytest
import torch

import route_case as rc
from test_gpu_fp8 import DT, _product_close, _wild

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    import sidekit_amd
    return sidekit_amd.default_engine()


def _values(m):
    return m.values().double().cpu().numpy()


def _operands(M, N, K, dtype, seed):
    a, _ = _wild((M, K), "bf16", seed)
    b, _ = _wild((N, K), "bf16", seed + 1)
    if dtype == "f16":
        a, b = a / 512, b / 512                              # results inside float16
    return a.cuda(), b.cuda()


# 256 x 128 with three stages (float32) or 256 x 256 (bf16, f16); 10 row tiles and a last one of 100 (half a tile) or 140
@pytest.mark.parametrize("M", [2660, 2700])
@pytest.mark.parametrize("dtype,K", [("f32", 1500), ("f32", 1664), ("bf16", 1200), ("bf16", 1536), ("f16", 1300)])
def test_large_tiles(eng, M, dtype, K):
    N = 3100
    a, b = _operands(M, N, K, dtype, K)
    A, B = eng.fp8_rows(a), eng.fp8_tiles(b)
    out = torch.full((M + 1, N), 5.0, dtype=DT[dtype], device="cuda")
    eng.gemm_fp8(A, B, out=out[:M])
    _product_close(out[:M], _values(A), _values(B))
    assert (out[M] == 5.0).all()
    old = out[:M].double().cpu().numpy()
    eng.gemm_fp8(A, B, out=out[:M], accumulate=True)
    va, vb = _values(A), _values(B)
    u = rc.U32 * (K + 1) + (2.0 ** -10 if dtype != "f32" else 0.0)      # as in _product_close
    ref, mag = va @ vb.T + old, np.abs(va) @ np.abs(vb).T + np.abs(old)
    tol = u * mag + rc.half_step(DT[dtype]) * np.abs(ref) + (2.0 ** -25 if dtype == "f16" else 0.0)
    assert (np.abs(out[:M].double().cpu().numpy() - ref) <= tol).all()


# few rows, one row tile after another in registers, 128 x 128 in slabs and not, 256 x 256
@pytest.mark.parametrize("M,N,K", [(1, 200, 700), (16, 70, 1300), (40, 4100, 700), (64, 300, 2000), (130, 140, 700), (300, 2700, 1100),
                                   (2660, 3100, 1200)])
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("fa,fb", [("e5m2", "e4m3"), ("e4m3", "e5m2"), ("e5m2", "e5m2")])
def test_e5m2_on_the_8_bit_instructions(eng, M, N, K, dtype, fa, fb):
    a, b = _operands(M, N, K, dtype, M)
    A, B = eng.fp8_rows(a, fa), eng.fp8_tiles(b, fb)
    _product_close(eng.gemm_fp8(A, B, dtype=DT[dtype]), _values(A), _values(B))


@pytest.mark.parametrize("M", [1, 5, 16, 17, 33, 64])
@pytest.mark.parametrize("a_type", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_float_rows_on_the_way(eng, M, a_type, dtype):
    """a float A gives the bits of its fp8_rows, in whatever type it is and in rows apart"""
    N, K = 200, 1157
    a, b = _operands(M, N, K, "f16", M)
    a = a.to(DT[a_type])
    B = eng.fp8_tiles(b)
    want = eng.gemm_fp8(eng.fp8_rows(a), B, dtype=DT[dtype])
    assert torch.equal(eng.gemm_fp8(a, B, dtype=DT[dtype]), want)
    wide = torch.full((M, K + 9), 1e4, device="cuda").to(DT[a_type])
    wide[:, 3:K + 3] = a
    assert torch.equal(eng.gemm_fp8(wide[:, 3:K + 3], B, dtype=DT[dtype]), want)
    _product_close(want, _values(eng.fp8_rows(a)), _values(B))


@pytest.mark.parametrize("a_type", ["f32", "f16"])
@pytest.mark.parametrize("T,k,E", [(8, 4, 64), (300, 2, 4), (700, 2, 2)])
def test_float_rows_of_experts(eng, a_type, T, k, E):
    """16, 128 and 256 rows a tile"""
    N, K = 140, 700
    r = np.random.RandomState(T)
    ids = torch.from_numpy(r.randint(-1, E, (T, k)).astype(np.int32)).cuda()
    a, b = _operands(T, E * N, K, "f16", T)
    a = a.to(DT[a_type])
    W, plan = eng.fp8_tiles(b.view(E, N, K)), eng.route_plan(ids, E)
    n = int(plan.offsets[-1])
    for dtype in ("f32", "bf16"):
        got = eng.gemm_fp8_experts(a, W, plan, dtype=DT[dtype])
        assert torch.equal(got[:n], eng.gemm_fp8_experts(eng.fp8_rows(a), W, plan, dtype=DT[dtype])[:n])


COUNTS = [1124, 1200, 0, 676, 128, 129]         # last tiles of 100, 176, 164, 128 and 129 rows of 256


@pytest.mark.parametrize("dtype,fmt,by_token", [("f32", "e4m3", True), ("f32", "e5m2", False), ("bf16", "e4m3", True),
                                                ("bf16", "e5m2", True), ("f16", "e5m2", False)])
def test_experts_with_long_sums(eng, dtype, fmt, by_token):
    E, k, N, K = len(COUNTS), 2, 700, 1500
    r = np.random.RandomState(7)
    ids = np.repeat(np.arange(E), COUNTS).astype(np.int32)
    ids = np.concatenate([ids, np.full(-ids.size % k + 2 * k, -1, dtype=np.int32)])
    r.shuffle(ids)
    ids = ids.reshape(-1, k)
    T = ids.shape[0]
    a, b = _operands(T, E * N, K, dtype, 3)
    W, plan = eng.fp8_tiles(b.view(E, N, K)), eng.route_plan(torch.from_numpy(ids).cuda(), E)
    assert plan.more_rows == 256
    pair, expert, _ = rc.plan(ids, E)
    if by_token:
        A = eng.fp8_rows(a, fmt)
        va = _values(A)[pair // k]
    else:
        apart = torch.zeros(T * k, K, dtype=a.dtype, device="cuda")
        apart[:pair.size] = a[torch.from_numpy(pair // k).cuda()]
        A = eng.fp8_rows(apart, fmt)
        va = _values(A)[:pair.size]
    rows = eng.gemm_fp8_experts(A, W, plan, dtype=DT[dtype])
    vw = _values(W)
    for e in range(E):
        m = expert == e
        if m.any():
            _product_close(rows[torch.from_numpy(np.flatnonzero(m)).cuda()], va[m], vw[e])


# 256 x 128 with three stages: more than ten blocks an expert on average and tiles for half of the GPU
@pytest.mark.parametrize("fa,fb", [("e5m2", "e4m3"), ("e4m3", "e4m3")])
@pytest.mark.parametrize("N", [600, 700])       # row tiles of 88 and 188
def test_weight_gradient_with_long_sums(eng, fa, fb, N):
    T, k, E, K = 3000, 2, 3, 2000
    r = np.random.RandomState(9)
    ids = r.choice(E + 1, (T, k), p=[0.55, 0.3, 0.1, 0.05]).astype(np.int32)
    ids[ids == E] = -1
    x, _ = _wild((T, K), "bf16", 1)
    dy, _ = _wild((T, N), "bf16", 2)
    w = torch.from_numpy(r.rand(T, k)).float()
    plan = eng.route_plan(torch.from_numpy(ids).cuda(), E)
    assert plan.max_tiles // E > 10
    A = eng.fp8_columns(dy.cuda(), fa, plan=plan, weights=w.cuda())
    B = eng.fp8_columns(x.cuda(), fb, plan=plan)
    dw = eng.gemm_fp8_experts_wgrad(A, B, plan)
    first = plan.first.cpu().numpy()
    va, vb = _values(A), _values(B)
    for e in range(E):
        sl = slice(first[e] * 128, first[e + 1] * 128)
        _product_close(dw[e], va[:, sl], vb[:, sl])
    old = dw.clone()
    eng.gemm_fp8_experts_wgrad(A, B, plan, out=dw, accumulate=True)
    assert torch.equal(dw, 2 * old)


@pytest.mark.parametrize("M,N", [(3, 60), (16, 4200), (40, 300), (130, 140), (2660, 3100)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("fmt", ["e4m3", "e5m2"])
def test_nan_and_infinities_stay_in_their_row(eng, M, N, dtype, fmt):
    """on every kernel: a NaN (or infinity, which e4m3 has none of) leaves no number in its row and every number in the others"""
    K = 1450
    a = torch.rand(M, K, generator=torch.Generator().manual_seed(M)).cuda() + 0.5
    b = torch.rand(N, K, generator=torch.Generator().manual_seed(N)).cuda() + 0.5       # no zeros: infinity times 0 is NaN
    rows = torch.zeros(M, dtype=torch.bool)
    rows[[1, M - 1]] = True
    clean = eng.gemm_fp8(eng.fp8_rows(a, fmt), eng.fp8_tiles(b, fmt), dtype=DT[dtype])
    a[1, K - 1], a[M - 1, 700] = float("nan"), float("inf")
    got = eng.gemm_fp8(eng.fp8_rows(a, fmt), eng.fp8_tiles(b, fmt), dtype=DT[dtype])
    assert torch.isnan(got[1]).all() and not torch.isfinite(got[M - 1]).any()
    if fmt == "e5m2" and M > 2:
        assert (got[M - 1] == float("inf")).all()
    assert torch.equal(got[(~rows).cuda()], clean[(~rows).cuda()])
    # and of B in their column
    b[N - 1, 0] = float("nan")
    other = eng.gemm_fp8(eng.fp8_rows(a, fmt), eng.fp8_rows(b, fmt), dtype=DT[dtype])
    assert torch.isnan(other[:, N - 1]).all() and torch.isfinite(other[(~rows).cuda()][:, :N - 1]).all()


@pytest.mark.parametrize("M", [1, 16, 40, 300])
@pytest.mark.parametrize("every", [2, 4, 8, 16, 32, 64])
@pytest.mark.parametrize("cancel", [False, True])
def test_small_products_beside_large_ones(eng, M, every, cancel):
    """the loss of the 8-bit instructions at its worst stays inside its bound, 2^-10 of the sum of the products' magnitudes
    (see _product_close); float32 results lose nothing: sums of multiples of 2^-14 below 2^10 are exact"""
    N, K = 140, 1024
    k = torch.arange(K)
    a = torch.where(k % every == 0, 1.0, 2.0 ** -7).repeat(M, 1)
    if cancel:
        a[:, (k % (2 * every)) == every] = -1.0              # the large products add up to nothing
    b = torch.where(k % every == 0, 1.0, 2.0 ** -7).repeat(N, 1)
    A, B = eng.fp8_rows(a.cuda()), eng.fp8_rows(b.cuda())
    ref = a.double() @ b.double().t()
    mag = a.abs().double() @ b.double().t()
    assert torch.equal(eng.gemm_fp8(A, B, dtype=torch.float32).double().cpu(), ref)
    for dtype in (torch.bfloat16, torch.float16):
        c = eng.gemm_fp8(A, B, dtype=dtype).double().cpu()
        tol = (2.0 ** -10 + rc.U32 * K) * mag + rc.half_step(dtype) * ref.abs() + 2.0 ** -25
        assert ((c - ref).abs() <= tol).all()
