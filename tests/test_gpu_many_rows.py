"""More rows than one launch can have workgroups for (fewer than 2^32 threads along x): every row has its result."""
import pytest
import torch

pytestmark = pytest.mark.gpu
GROUPS = 1 << 24                # workgroups of 256 threads


@pytest.fixture(scope="module")
def eng():
    import sidekit_amd
    return sidekit_amd.default_engine()


def _again(small, rows):
    """the rows of `small` over and over"""
    return small.repeat(-(-rows // small.shape[0]), *([1] * (small.dim() - 1)))[:rows]


def _logits(E, dtype, seed):
    return torch.randn(4099, E, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


@pytest.mark.parametrize("dtype,renorm,per_group", [(torch.bfloat16, True, 16),      # 16 lanes a row
                                                    (torch.float64, False, 4)])      # a wave a row
def test_route(eng, dtype, renorm, per_group):
    T, E = GROUPS * per_group + 37, 4
    small = _logits(E, dtype, 1)
    ids, w = eng.route(small, 1, renorm=renorm)
    got, gw = eng.route(_again(small, T), 1, renorm=renorm)
    assert torch.equal(got, _again(ids, T)) and torch.equal(gw, _again(w, T))


@pytest.mark.parametrize("dtype,per_group", [(torch.bfloat16, 16), (torch.float64, 4)])
def test_route_backward(eng, dtype, per_group):
    T, E = GROUPS * per_group + 37, 4
    small = _logits(E, dtype, 2)
    ids, w = eng.route(small, 2)
    g = torch.randn(4099, 2, generator=torch.Generator().manual_seed(3)).cuda()
    dx = eng.route_backward(small, ids, g)
    assert float(dx.abs().sum()) > 0
    got = eng.route_backward(_again(small, T), _again(ids, T), _again(g, T))
    assert torch.equal(got, _again(dx, T))


def test_combine(eng):
    """a token a workgroup: rows of more than 128 threads"""
    T, N = GROUPS + 3, 1032
    rows = torch.randn(4099, N, generator=torch.Generator().manual_seed(4)).bfloat16().cuda()
    pos = _again(torch.arange(4099, dtype=torch.int32, device="cuda"), T)
    w = torch.full((T,), 1.0, device="cuda")
    out = torch.empty(T, N, dtype=torch.bfloat16, device="cuda")
    eng._check(eng.lib.skm_route_combine(eng.ctx, rows.data_ptr(), 1, pos.data_ptr(), w.data_ptr(), T, 1, N,
                                         out.data_ptr(), 1, eng._raw_stream()))
    step = 4099 * 256
    for t in range(0, T, step):
        part = out[t:t + step]
        assert torch.equal(part, _again(rows, part.shape[0]))


def test_combine_of_short_rows_and_its_gradient(eng):
    T, k, N = GROUPS * 2 + 5, 2, 1              # more pairs than a wave each has room for in one launch
    r = torch.Generator().manual_seed(5)
    ids = _again(torch.randint(0, 2, (4099, k), generator=r).int().cuda(), T)
    plan = eng.route_plan(ids, 2)
    rows = torch.randn(plan.n, N, device="cuda")
    dout = torch.randn(T, N, device="cuda")
    dw = eng.route_combine_backward(rows, dout, plan)
    # one product a pair
    assert torch.equal(dw, rows[:, 0][plan.pos.long()] * dout)
    w = torch.ones(T, k, device="cuda")
    out = eng.route_combine(rows, w, plan)
    both = rows[:, 0][plan.pos.long()]
    assert torch.equal(out[:, 0], both[:, 0] + both[:, 1])


def test_fp8_rows(eng):
    M = GROUPS * 16 + 19                        # blocks of 128, 16 a workgroup
    small = _logits(1, torch.bfloat16, 6)
    want = eng.fp8_rows(small)
    got = eng.fp8_rows(_again(small, M))
    assert torch.equal(got.s, _again(want.s, M))
    step = 4099 * 4096
    for m in range(0, M, step):
        part = got.q[m:m + step]
        assert torch.equal(part, _again(want.q, part.shape[0]))
