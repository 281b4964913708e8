"""What the routing and 8-bit product entry points refuse, on the CPU: the C-ABI's argument checks (they come before any
call of the runtime) and those of the engine's methods, on an engine whose device is the CPU."""
import ctypes
import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
import sidekit_amd as sk        # noqa: E402

ARG, WORKSPACE, UNSUPPORTED = -1, -3, -4


@pytest.fixture(scope="module")
def lib():
    return sk.load_library()


@pytest.fixture(scope="module")
def ctx():
    return ctypes.create_string_buffer(1024)        # never looked at by a refused call


class _CpuEngine(sk.HipEngine):
    def __init__(self, lib):
        self.torch, self.lib, self.device = torch, lib, torch.device("cpu")
        self.ctx = None                              # the library refuses a call without a context
        self._dt_codes = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2, torch.float64: 3}

    def _stream(self):
        return None

    def _raw_stream(self):
        return None

    def close(self):
        pass


@pytest.fixture(scope="module")
def eng(lib):
    return _CpuEngine(lib)


P = ctypes.c_void_p(0x1000)     # some address that is never followed


def _route(lib, ctx, **kw):
    a = dict(x=P, dtype=0, T=4, E=8, ldx=8, k=2, scores=0, bias=None, groups=1, group_k=1, group_top=2, renorm=1,
             scale=1.0, ids=P, w=P)
    a.update(kw)
    return lib.skm_route(ctx, a["x"], a["dtype"], a["T"], a["E"], a["ldx"], a["k"], a["scores"], a["bias"], a["groups"],
                         a["group_k"], a["group_top"], a["renorm"], a["scale"], a["ids"], a["w"], None)


@pytest.mark.parametrize("kw,rc", [
    (dict(x=None), ARG), (dict(ids=None), ARG), (dict(w=None), ARG), (dict(dtype=7), ARG), (dict(T=-1), ARG),
    (dict(E=0), ARG), (dict(ldx=7), ARG), (dict(k=0), ARG), (dict(k=9), ARG), (dict(scores=2), ARG),
    (dict(groups=3), ARG), (dict(groups=0), ARG), (dict(groups=4, group_k=0), ARG), (dict(groups=4, group_k=5), ARG),
    (dict(groups=4, group_k=1, k=3), ARG), (dict(group_top=3), ARG), (dict(E=5000, ldx=5000), UNSUPPORTED),
    (dict(E=128, ldx=128, k=65), UNSUPPORTED), (dict(E=130, ldx=130, groups=65, group_k=65), UNSUPPORTED),
    (dict(T=0, x=None, ids=None, w=None), 0)])
def test_route_refusals(lib, ctx, kw, rc):
    assert _route(lib, ctx, **kw) == rc
    if rc:
        assert b"skm_route" in lib.skm_last_error()


def test_route_without_context(lib):
    assert _route(lib, None) == ARG


@pytest.mark.parametrize("kw,rc", [(dict(dx=None), ARG), (dict(ids=None), ARG), (dict(g=None), ARG), (dict(k=9), ARG),
                                   (dict(ldx=3), ARG), (dict(scores=-1), ARG), (dict(E=4097, ldx=4097), UNSUPPORTED),
                                   (dict(T=0), 0)])
def test_route_backward_refusals(lib, ctx, kw, rc):
    a = dict(x=P, dtype=0, T=4, E=8, ldx=8, k=2, scores=0, ids=P, g=P, dx=P)
    a.update(kw)
    assert lib.skm_route_backward(ctx, a["x"], a["dtype"], a["T"], a["E"], a["ldx"], a["k"], a["scores"], 1, 1.0, a["ids"],
                                  a["g"], a["dx"], None) == rc


@pytest.mark.parametrize("kw,rc", [(dict(ids=None), ARG), (dict(E=0), ARG), (dict(n=-1), ARG), (dict(E=4097), UNSUPPORTED),
                                   (dict(n=1 << 31), UNSUPPORTED), (dict(n=1 << 20, ws_bytes=8), WORKSPACE),
                                   (dict(n=1 << 20, ws=None, ws_bytes=1 << 40), WORKSPACE),
                                   (dict(more=P, more_rows=16, more_count=None), ARG),
                                   (dict(more=P, more_rows=32, more_count=P), ARG),
                                   (dict(more=ctypes.c_void_p(0x1008), more_rows=16, more_count=P), ARG)])
def test_route_plan_refusals(lib, ctx, kw, rc):
    a = dict(ids=P, n=64, E=8, ws=P, ws_bytes=0, more=None, more_rows=0, more_count=None)
    a.update(kw)
    assert lib.skm_route_plan(ctx, a["ids"], a["n"], a["E"], P, P, P, P, P, a["more_rows"], a["more"],
                              a["more_count"], a["ws"],
                              a["ws_bytes"], None) == rc


def test_plan_sizes(lib):
    # every expert adds less than one tile to its full ones, and there are no more tiles than pairs
    for n, E, rows in ((0, 4, 128), (1, 4, 128), (5, 4, 16), (1000, 7, 128), (4096, 4096, 16)):
        worst = 0
        left = n
        for e in range(E):                           # E - 1 experts with one pair, the last with the others
            c = min(left, 1) if e < E - 1 else left
            left -= c
            worst += -(-c // rows)
        assert lib.skm_route_plan_tiles(n, E, rows) >= worst
    assert lib.skm_route_plan_tiles(-1, 4, 128) == 0
    assert lib.skm_fp8_row_bytes(1) == 128 and lib.skm_fp8_row_bytes(129) == 256 and lib.skm_fp8_row_bytes(0) == 0
    assert lib.skm_fp8_scale_bytes(128) == 4 and lib.skm_fp8_scale_bytes(513) == 8


def test_combine_refusals(lib, ctx):
    f = lib.skm_route_combine
    assert f(ctx, P, 0, P, P, 4, 2, 0, P, 0, None) == ARG
    assert f(ctx, None, 0, P, P, 4, 2, 8, P, 0, None) == ARG
    assert f(ctx, P, 0, P, P, 4, 0, 8, P, 0, None) == ARG
    assert f(ctx, P, 1, P, P, 0, 2, 8, P, 2, None) == 0
    g = lib.skm_route_combine_backward
    assert g(ctx, P, 0, P, None, 0, 4, 2, 8, P, None) == ARG
    assert g(ctx, P, 0, P, P, 0, 4, 2, 8, None, None) == ARG


def test_fp8_refusals(lib, ctx):
    assert lib.skm_fp8_rows(ctx, P, 3, 4, 8, 8, 0, P, P, None) == ARG          # float64
    assert lib.skm_fp8_rows(ctx, P, 0, 4, 8, 7, 0, P, P, None) == ARG
    assert lib.skm_fp8_rows(ctx, P, 0, 4, 0, 8, 0, P, P, None) == ARG
    assert lib.skm_fp8_rows(ctx, P, 0, 4, 8, 8, 2, P, P, None) == ARG
    assert lib.skm_fp8_rows(ctx, P, 0, 4, 8, 8, 0, None, P, None) == ARG
    assert lib.skm_fp8_rows(ctx, None, 0, 0, 8, 8, 0, None, None, None) == 0
    assert lib.skm_fp8_tiles(ctx, P, 0, 1, 8, 8, 8, 64, 0, P, P, P, None, None) == ARG
    assert lib.skm_fp8_tiles(ctx, P, 0, 1, 0, 8, 8, 64, 0, P, P, None, None, None) == ARG
    assert lib.skm_fp8_columns(ctx, P, 0, 8, 8, 8, 0, P, None, 4, P, 2, None, P, P, None) == ARG
    assert lib.skm_fp8_columns(ctx, P, 0, 8, 8, 8, 0, None, None, 0, None, 0, P, P, P, None) == ARG
    gemm = lib.skm_gemm_fp8
    odd = ctypes.c_void_p(0x1004)
    assert gemm(ctx, P, P, 0, -1, 0, P, P, 0, 8, 8, 0, P, 0, 8, 0, None, 0, None) == ARG          # no K
    assert gemm(ctx, P, P, 0, -1, 0, P, P, 0, 8, 8, 8, P, 3, 8, 0, None, 0, None) == ARG          # float64 result
    assert gemm(ctx, P, P, 2, -1, 0, P, P, 0, 8, 8, 8, P, 0, 8, 0, None, 0, None) == ARG          # format
    assert gemm(ctx, P, P, 0, -1, 0, P, P, 0, 8, 8, 8, P, 0, 7, 0, None, 0, None) == ARG          # ldc < N
    assert gemm(ctx, P, None, 0, -1, 0, P, P, 0, 8, 8, 8, P, 0, 8, 0, None, 0, None) == ARG       # no scales
    assert gemm(ctx, P, P, 0, 3, 8, P, P, 0, 8, 8, 8, P, 0, 8, 0, None, 0, None) == ARG           # float64 A
    assert gemm(ctx, P, P, 0, 0, 7, P, P, 0, 8, 8, 8, P, 0, 8, 0, None, 0, None) == ARG           # rows overlap
    assert gemm(ctx, P, P, 0, 0, 8, P, P, 0, 99, 8, 8, P, 0, 8, 0, None, 0, None) == WORKSPACE
    assert gemm(ctx, P, P, 0, 0, 8, P, P, 0, 99, 8, 8, P, 0, 8, 0, odd, 1 << 20, None) == WORKSPACE
    assert gemm(ctx, odd, P, 0, -1, 0, P, P, 0, 8, 8, 8, P, 0, 8, 0, None, 0, None) == ARG        # alignment
    assert gemm(ctx, P, P, 0, -1, 0, odd, P, 0, 8, 8, 8, P, 0, 8, 0, None, 0, None) == ARG
    assert gemm(ctx, P, P, 0, -1, 0, P, P, 0, 0, 8, 8, P, 0, 8, 0, None, 0, None) == 0
    assert lib.skm_gemm_fp8_workspace_bytes(ctx, 99, 8, 8, 0) == 0
    assert lib.skm_gemm_fp8_workspace_bytes(ctx, 99, 8, 8, 1) >= 99 * (128 + 4)
    ex = lib.skm_gemm_fp8_experts
    assert ex(ctx, P, P, 0, -1, 0, 4, P, P, 0, 0, 8, 8, P, 2, 8, P, P, 0, None, None, P, 0, None, 0, None) == ARG     # E
    assert ex(ctx, P, P, 0, -1, 0, 4, P, P, 0, 4, 8, 8, None, 2, 8, P, P, 0, None, None, P, 0, None, 0, None) == ARG  # no pairs
    assert ex(ctx, P, P, 0, -1, 0, 5, P, P, 0, 4, 8, 8, P, 2, 8, P, P, 0, None, None, P, 0, None, 0, None) == ARG     # 5 x 2 != 8
    assert ex(ctx, P, P, 0, -1, 0, 4, P, P, 0, 4, 8, 8, P, 0, 8, P, P, 0, None, None, P, 0, None, 0, None) == ARG
    assert ex(ctx, P, P, 0, -1, 0, 4, P, P, 0, 4, 8, 8, P, 2, 8, P, P, 16, P, None, P, 0, None, 0, None) == ARG        # no count
    assert ex(ctx, P, None, 0, 0, 8, 4, P, P, 0, 4, 8, 8, P, 2, 8, P, P, 0, None, None, P, 0, None, 0, None) == WORKSPACE
    assert lib.skm_gemm_fp8_experts_wgrad(ctx, P, P, 0, P, P, 0, 4, 8, 8, P, 2, None, 0, None) == ARG
    assert lib.skm_gemm_fp8_experts_wgrad(ctx, P, P, 0, P, P, 0, 70000, 8, 8, P, 2, P, 0, None) == ARG


def _refused(f, *a, **kw):
    with pytest.raises(sk.SkmError):
        f(*a, **kw)


def test_engine_refusals(eng):
    x = torch.zeros(4, 8)
    _refused(eng.route, x.t(), 2)                                   # rows not contiguous
    _refused(eng.route, torch.zeros(4), 2)
    _refused(eng.route, x.to(torch.int32), 2)
    _refused(eng.route, x, 0)
    _refused(eng.route, x, -1)
    _refused(eng.route, x, 2, scores="top")
    _refused(eng.route, x, 2, bias=torch.zeros(7))
    _refused(eng.route, x, 2, bias=torch.zeros(8, dtype=torch.float64))
    _refused(eng.route, x[:, ::2], 2)
    ids, g = torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2)
    _refused(eng.route_backward, x, ids.long(), g)
    _refused(eng.route_backward, x, ids, g[:3])
    _refused(eng.route_backward, x, ids, g.double())
    _refused(eng.route_plan, ids.long(), 8)
    _refused(eng.route_plan, ids, 0)
    _refused(eng.route_plan, ids.t(), 8)
    _refused(eng.fp8_rows, x.double())
    _refused(eng.fp8_rows, x, "e3m4")
    _refused(eng.fp8_rows, x[:, :0])
    _refused(eng.fp8_tiles, x.t())
    _refused(eng.fp8_columns, x, weights=g)
    A, B = sk.Fp8Matrix(eng, (4,), 8, "e4m3"), sk.Fp8Matrix(eng, (6,), 9, "e4m3")
    _refused(eng.gemm_fp8, A, B)                                    # K differs
    _refused(eng.gemm_fp8, A, x)
    C = sk.Fp8Matrix(eng, (6,), 8, "e4m3")
    _refused(eng.gemm_fp8, A, C, accumulate=True)
    _refused(eng.gemm_fp8, A, C, out=torch.zeros(4, 5))
    _refused(eng.gemm_fp8, A, C, out=torch.zeros(6, 4).t())
    _refused(eng.gemm_fp8, A, C, dtype=torch.float64)
    plan = sk.RoutePlan(eng, 4, 2, 3)
    W = sk.Fp8Matrix(eng, (3, 6), 8, "e4m3")
    _refused(eng.gemm_fp8_experts, A, C, plan)
    _refused(eng.gemm_fp8_experts, sk.Fp8Matrix(eng, (5,), 8, "e4m3"), W, plan)
    _refused(eng.gemm_fp8_experts, A, sk.Fp8Matrix(eng, (2, 6), 8, "e4m3"), plan)
    _refused(eng.gemm_fp8_experts_wgrad, A, C, plan)                # not from fp8_columns with the plan
    _refused(eng.route_combine, torch.zeros(7, 6), g, plan)
    _refused(eng.route_combine, torch.zeros(8, 6), g[:3], plan)
    _refused(eng.route_combine_backward, torch.zeros(8, 6), torch.zeros(4, 5), plan)
    # a valid call reaches the library, which wants a context
    _refused(eng.route, x, 2)


@pytest.mark.parametrize("T,k,E", [(0, 2, 5), (1, 1, 1), (7, 3, 4), (8, 4, 64), (300, 2, 4), (5000, 3, 130)])
def test_plan_layout(eng, lib, T, k, E):
    """the plan's tensors do not overlap, fit and are aligned as the library wants them"""
    p = sk.RoutePlan(eng, T, k, E)
    n = T * k
    assert p.max_tiles == lib.skm_route_plan_tiles(n, E, 128)
    if p.more_rows:
        assert p._view("more_tiles").numel() == 4 * lib.skm_route_plan_tiles(n, E, p.more_rows)
    spans = []
    for name in ("offsets", "pair", "pos", "first", "tiles", "more_tiles", "more_count"):
        v = p._view(name)
        assert v.numel() == 0 or v.data_ptr() == p._ptr(name)
        if name in ("tiles", "more_tiles"):
            assert (p._ptr(name) - p._base) % 16 == 0
        spans.append((p._at[name], p._at[name] + v.numel()))
    spans.sort()
    assert all(a[1] <= b[0] for a, b in zip(spans, spans[1:])) and spans[-1][1] <= p._buf.numel()
    assert p._ptr("tile_count") == p._ptr("first") + 4 * E


def test_values_of_a_matrix(eng):
    m = sk.Fp8Matrix(eng, (2,), 130, "e4m3")
    m.q.zero_()
    m.s.fill_(127)
    m.q[0, 0], m.q[1, 129] = 0x38, 0xB8          # 1 and -1
    m.s[1, 1] = 130
    v = m.values()
    assert tuple(v.shape) == (2, 130) and float(v[0, 0]) == 1.0 and float(v[1, 129]) == -8.0
    assert float(v.abs().sum()) == 9.0
