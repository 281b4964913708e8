"""The router and its experts' products run together, as a user's program runs them: the components of a mixture chosen per
frame and their linear transforms applied, a training step of it, on other streams, captured into graphs, with nothing to do."""
import numpy as np
import pytest
import torch

import route_case as rc

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng():
    import sidekit_amd
    return sidekit_amd.default_engine()


def _forward(eng, x, logits, W, k, dtype=torch.float32):
    ids, w = eng.route(logits, k)
    plan = eng.route_plan(ids, W.shape[0])
    rows = eng.gemm_fp8_experts(x, W, plan, dtype=dtype)
    return eng.route_combine(rows, w, plan), ids, w, plan, rows


def _step(eng, x, logits, w, dout, k):
    """a training step: out, dx, dw, dlogits"""
    W, Wt = eng.fp8_tiles(w, transposed=True)
    out, ids, weights, plan, rows = _forward(eng, eng.fp8_rows(x), logits, W, k)
    dx = eng.route_combine(eng.gemm_fp8_experts(eng.fp8_rows(dout), Wt, plan, dtype=torch.float32), weights, plan)
    dweights = eng.route_combine_backward(rows, dout, plan)
    dlogits = eng.route_backward(logits, ids, dweights)
    dw = eng.gemm_fp8_experts_wgrad(eng.fp8_columns(dout, plan=plan, weights=weights), eng.fp8_columns(x, plan=plan), plan)
    return out, dx, dw, dlogits, ids, weights


def test_components_of_a_mixture(eng):
    """posterior-weighted transforms of frames by the 4 best components: log-probabilities of the mixture's kernels, chosen,
    weighted and applied"""
    from oracle import sidekit_ref as orc
    C, D, O, T, k = 64, 60, 48, 777, 4
    gmm = orc.random_gmm(C, D, seed=3)
    cep = orc.synth_frames(T, dim=D, seed=4)
    X = eng.upload_frames(cep)
    lp = eng.logprob(X, eng.pack(gmm.w, gmm.mu, gmm.invcov))
    w = torch.randn(C, O, D, generator=torch.Generator().manual_seed(5)).cuda() / D ** 0.5
    W = eng.fp8_tiles(w)
    y, ids, weights, plan, _ = _forward(eng, X, lp, W, k)
    rids, rw, _ = rc.route(lp.cpu().numpy(), k)
    np.testing.assert_array_equal(ids.cpu().numpy(), rids)
    # posteriors of all components, cut to the k best and renormalised
    pp, _ = eng.row_logsumexp(lp)
    best = torch.gather(pp, 1, ids.long())
    assert torch.allclose(weights.double(), best / best.sum(1, keepdim=True), rtol=1e-5, atol=1e-12)
    xq, wq = eng.fp8_rows(X).values().double().cpu().numpy(), W.values().double().cpu().numpy()
    ref, mag = np.zeros((T, O)), np.zeros((T, O))
    for j in range(k):
        part = np.einsum("tod,td->to", wq[rids[:, j]], xq)
        ref += rw[:, j, None] * part
        mag += rw[:, j, None] * np.einsum("tod,td->to", np.abs(wq[rids[:, j]]), np.abs(xq))
    # D exact products summed in float32, weights good to some 2^-20 (exponents of up to 88), k terms
    assert (np.abs(y.double().cpu().numpy() - ref) <= (rc.U32 * (D + k + 4) + 2.0 ** -16) * mag).all()


def test_training_step(eng):
    T, E, k, N, K = 210, 6, 3, 70, 150
    g = torch.Generator().manual_seed(1)
    x, logits = torch.randn(T, K, generator=g), torch.randn(T, E, generator=g)
    w, dout = torch.randn(E, N, K, generator=g) / K ** 0.5, torch.randn(T, N, generator=g)
    logits[5] = float("-inf")                                # a token without experts
    out, dx, dw, dlogits, ids, weights = [v.cpu() for v in _step(eng, x.cuda(), logits.cuda(), w.cuda(), dout.cuda(), k)]
    xd, wd, dd, ld = x.double().numpy(), w.double().numpy(), dout.double().numpy(), logits.double().numpy()
    rids, rw, _ = rc.route(ld, k)
    np.testing.assert_array_equal(ids.numpy(), rids)
    xq = rc.fp8_blocks(xd, "e4m3", 1, 128)[0]
    dq = rc.fp8_blocks(dd, "e4m3", 1, 128)[0]
    wq = np.stack([rc.fp8_blocks(wd[e], "e4m3", 128, 128)[0] for e in range(E)])
    tol = rc.U32 * (max(T * k, K, N) + 64)

    def near(got, ref, mag):
        assert (np.abs(got.double().numpy() - ref) <= tol * mag + 1e-30).all()

    ro, rdx, mo, mdx = (np.zeros(s) for s in ((T, N), (T, K), (T, N), (T, K)))
    rdw, mdw, rg, mg = np.zeros((E, N, K)), np.zeros((E, N, K)), np.zeros((T, k)), np.zeros((T, k))
    for e in range(E):
        t, j = np.nonzero(rids == e)
        s = weights.double().numpy()[t, j][:, None]
        ro[t] += s * (xq[t] @ wq[e].T)
        mo[t] += s * (np.abs(xq[t]) @ np.abs(wq[e]).T)
        rdx[t] += s * (dq[t] @ wq[e])
        mdx[t] += s * (np.abs(dq[t]) @ np.abs(wq[e]))
        rg[t, j] = ((xq[t] @ wq[e].T) * dd[t]).sum(1)
        mg[t, j] = ((np.abs(xq[t]) @ np.abs(wq[e]).T) * np.abs(dd[t])).sum(1)
        a = rc.fp8_blocks((dout.numpy()[t] * weights.numpy()[t, j][:, None]).astype(np.float64), "e4m3", 128, 1)[0]
        b = rc.fp8_blocks(xd[t], "e4m3", 128, 1)[0]
        rdw[e], mdw[e] = a.T @ b, np.abs(a).T @ np.abs(b)
    near(out, ro, mo)
    near(dx, rdx, mdx)
    near(dw, rdw, mdw)
    rl, _ = rc.route_backward(ld, rids, rg)
    _, ml = rc.route_backward(ld, rids, mg)
    near(dlogits, rl, ml)
    assert (out[5] == 0).all() and (dx[5] == 0).all() and (dlogits[5] == 0).all()


def test_training_step_against_differences(eng):
    """The gradients of L = <out, dout> against central differences of the step's formula without 8-bit numbers, in float64.
    Every operand is off by at most 2^-4 of itself or, near zero, 2^-10 of its block's scale (448 2^e <= 2 max |block|, the
    smallest step of e4m3 2^-9 2^e): at most 2^-4 |v| + 2^-17 max |block| each, two operands a product."""
    T, E, k, N, K = 40, 4, 2, 20, 30
    g = torch.Generator().manual_seed(2)
    x, logits = torch.randn(T, K, generator=g), torch.randn(T, E, generator=g)
    w, dout = torch.randn(E, N, K, generator=g) / K ** 0.5, torch.randn(T, N, generator=g)
    _, dx, dw, dlogits, ids, _ = [v.cpu().double().numpy() for v in _step(eng, x.cuda(), logits.cuda(), w.cuda(), dout.cuda(), k)]
    xd, wd, dd, ld = x.double().numpy(), w.double().numpy(), dout.double().numpy(), logits.double().numpy()
    ids = ids.astype(int)

    def loss(xv, wv, lv):
        s = np.take_along_axis(lv, ids, 1)
        s = np.exp(s - s.max(1, keepdims=True))
        s /= s.sum(1, keepdims=True)
        y = np.einsum("tjnk,tk->tjn", wv[ids], xv)
        return (s[:, :, None] * y * dd[:, None, :]).sum()

    s = np.take_along_axis(ld, ids, 1)
    s = np.exp(s - s.max(1, keepdims=True))
    s /= s.sum(1, keepdims=True)
    off = lambda v: 2.0 ** -4 * np.abs(v) + 2.0 ** -17 * np.abs(v).max()     # noqa: E731
    r = np.random.RandomState(0)
    h = 1e-6
    for _ in range(20):
        t, c, e, n = r.randint(T), r.randint(K), r.randint(E), r.randint(N)
        for what, got, at in (("x", dx, (t, c)), ("w", dw, (e, n, c)), ("l", dlogits, (t, e))):
            p = {"x": xd, "w": wd, "l": ld}
            lo, hi = dict(p), dict(p)
            lo[what], hi[what] = p[what].copy(), p[what].copy()
            lo[what][at] -= h
            hi[what][at] += h
            num = (loss(hi["x"], hi["w"], hi["l"]) - loss(lo["x"], lo["w"], lo["l"])) / (2 * h)
            if what == "x":
                a, b = dd[t], wd[ids[t]][:, :, c]
                tol = (s[t][:, None] * (off(dd)[t][None] * np.abs(b) + np.abs(a)[None] * off(wd)[ids[t]][:, :, c]
                                        + off(dd)[t][None] * off(wd)[ids[t]][:, :, c])).sum()
            elif what == "w":
                tt, j = np.nonzero(ids == e)
                a, b = s[tt, j] * dd[tt, n], xd[tt, c]
                oa, ob = 2.0 ** -4 * np.abs(a) + 2.0 ** -17 * np.abs(dd).max(), off(xd)[tt, c]
                tol = (oa * np.abs(b) + np.abs(a) * ob + oa * ob).sum()
            else:
                # of each place's dweight, the products' errors, through the weights' gradient (twice its magnitude)
                y = (np.abs(dd[t])[None, :, None] * (off(wd)[ids[t]] * np.abs(xd[t]) + np.abs(wd[ids[t]]) * off(xd)[t]
                                                     + off(wd)[ids[t]] * off(xd)[t])).sum((1, 2))
                j = np.flatnonzero(ids[t] == e)
                tol = 0.0 if not j.size else float(s[t, j[0]] * (y[j[0]] + (s[t] * y).sum()))
            assert abs(num - got[at]) <= tol + 1e-6, (what, at, num, got[at], tol)


def _inputs(T, E, N, K, seed):
    g = torch.Generator().manual_seed(seed)
    return [v.cuda() for v in (torch.randn(T, K, generator=g), torch.randn(T, E, generator=g),
                               torch.randn(E, N, K, generator=g), torch.randn(T, N, generator=g))]


@pytest.mark.parametrize("T,E,k", [(5, 8, 2), (300, 4, 2), (3000, 3, 2)])
def test_graphs(eng, T, E, k):
    """two captured training steps, replayed in turn with new inputs and eager work between the replays"""
    N, K = 136, 264
    graphs = []
    for seed in (1, 2):
        held = _inputs(T, E, N, K, seed)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _step(eng, *held, k)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = _step(eng, *held, k)
        graphs.append((graph, held, got))
    for turn in range(3):
        want = []
        for i, (graph, held, got) in enumerate(graphs):
            new = _inputs(T, E, N, K, 10 * turn + i)
            want.append([v.clone() for v in _step(eng, *new, k)])        # eager, between the replays
            for h, v in zip(held, new):
                h.copy_(v)
            graph.replay()
        torch.cuda.synchronize()
        for (graph, held, got), w in zip(graphs, want):
            for a, b in zip(got, w):
                assert torch.equal(a, b)


def test_streams(eng):
    """two steps on two streams at once, and the same on the default one"""
    cases = [_inputs(700, 5, 130, 200, s) for s in (3, 4)]
    want = [[v.clone() for v in _step(eng, *c, 2)] for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        got = []
        for c, st in zip(cases, streams):
            with torch.cuda.stream(st):
                got.append(_step(eng, *c, 2))
        for st in streams:
            st.synchronize()
        for g, w in zip(got, want):
            assert all(torch.equal(a, b) for a, b in zip(g, w))


def test_nothing_to_do(eng):
    """no tokens; tokens without any expert"""
    out, dx, dw, dlogits, ids, w = _step(eng, *_inputs(0, 4, 20, 30, 1), 2)
    assert out.shape == (0, 20) and dx.shape == (0, 30) and dlogits.shape == (0, 4) and (dw == 0).all()
    x, logits, wt, dout = _inputs(9, 4, 20, 30, 1)
    out, dx, dw, dlogits, ids, w = _step(eng, x, torch.full_like(logits, float("-inf")), wt, dout, 2)
    assert (ids == -1).all() and (w == 0).all()
    assert all((v == 0).all() for v in (out, dx, dw, dlogits))


def test_far_offsets(eng):
    """logits, activations and results whose byte offsets pass 32 bits; the last rows against small calls on them"""
    T, E = 1200007, 1024                                     # 2.4 GB of bf16 logits each row 2 KB: more than 2^31 bytes
    x = torch.randn(4096, E, generator=torch.Generator().manual_seed(1)).bfloat16().cuda().repeat(T // 4096 + 1, 1)[:T]
    ids, w = eng.route(x, 4)
    lids, lw = eng.route(x[-5000:].contiguous(), 4)
    assert torch.equal(ids[-5000:], lids) and torch.equal(w[-5000:], lw)
    dx = eng.route_backward(x, ids, torch.ones_like(w), renorm=False)
    assert torch.equal(dx[-5000:], eng.route_backward(x[-5000:].contiguous(), lids, torch.ones_like(lw), renorm=False))
    del dx, ids, w
    M, K, N = 1200007, 4000, 24                              # 4.9 GB of 8-bit activations
    a = torch.empty(M, K, dtype=torch.bfloat16, device="cuda")
    a[:] = x.view(-1)[:K * 1000].view(1000, K).repeat(M // 1000 + 1, 1)[:M]
    B = eng.fp8_tiles(torch.randn(N, K, generator=torch.Generator().manual_seed(2)).cuda())
    A = eng.fp8_rows(a)
    c = eng.gemm_fp8(A, B)
    last = eng.gemm_fp8(a[-300:].contiguous(), B)
    # the same products; another kernel may add them in another order: two roundings to bf16 of sums that differ by 2^-9 at most
    assert torch.allclose(c[-300:].float(), last.float(), rtol=2.0 ** -7, atol=1e-2)
    assert torch.equal(A.q[-300:], eng.fp8_rows(a[-300:].contiguous()).q)
