"""Plain 64-bit forms of the routing and 8-bit product operators, for the tests (CPU, numpy / torch float64)."""
import numpy as np
import torch

U32 = 2.0 ** -24        # half a step of float32, relative


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def route(x, k, scores="softmax", bias=None, groups=1, group_k=None, group_top=2, renorm=True, scale=1.0):
    """x: float64 numpy [T, E].  Returns ids, weights, p."""
    T, E = x.shape
    group_k = groups if group_k is None else group_k
    ids = np.full((T, k), -1, dtype=np.int32)
    w = np.zeros((T, k))
    P = np.zeros((T, E))
    for t in range(T):
        row = x[t]
        on = row != -np.inf
        if bias is not None:
            on = on & (bias != -np.inf)
        bad = np.isnan(row).any() or (scores == "softmax" and (row == np.inf).any())
        if bad:
            w[t] = np.nan
            continue
        with np.errstate(over="ignore"):
            if scores == "softmax":
                m = row.max()
                p = np.exp(row - m) if np.isfinite(m) else np.zeros(E)
                p = p / p.sum() if p.sum() > 0 else p
            else:
                p = 1.0 / (1.0 + np.exp(-row))
        P[t] = p
        c = p + bias.astype(np.float64) if bias is not None else p
        order = c if bias is not None else row
        stay = on.copy()
        if groups > 1:
            per = E // groups
            score = np.full(groups, -np.inf)
            for g in range(groups):
                v = np.sort(c[g * per:(g + 1) * per][on[g * per:(g + 1) * per]])[::-1][:group_top]
                if v.size:
                    score[g] = v.sum()
            best = np.argsort(-score, kind="stable")[:group_k]
            keep = np.zeros(groups, dtype=bool)
            keep[best] = True
            stay &= np.repeat(keep, per)
        cand = np.flatnonzero(stay)
        cand = cand[np.argsort(-order[cand], kind="stable")][:k]
        ids[t, :cand.size] = cand
        if not cand.size:
            continue
        if renorm:
            xs = row[cand]
            if scores == "softmax":
                s = np.exp(xs - xs.max())
            else:
                lw = np.minimum(xs, 0) - np.log1p(np.exp(-np.abs(xs)))
                s = np.exp(lw - lw.max())
            w[t, :cand.size] = s / s.sum() * scale
        else:
            w[t, :cand.size] = p[cand] * scale
    return ids, w, P


def route_backward(x, ids, g, scores="softmax", renorm=True, scale=1.0):
    """(gradient of x, sum of the magnitudes of its terms) in float64, by automatic differentiation of the formula"""
    ok = (ids >= 0) & (ids < x.shape[1])
    ok &= np.take_along_axis(x, np.where(ok, ids, 0), 1) != -np.inf
    at = torch.from_numpy(np.where(ok, ids, 0).astype(np.int64))
    okt = torch.from_numpy(ok)
    xt = torch.from_numpy(x.copy()).requires_grad_(True)
    gt = torch.from_numpy(g.astype(np.float64))
    if scores == "softmax" and renorm:
        lp = xt                     # the row's log-sum-exp cancels
    elif scores == "softmax":
        lp = xt - torch.logsumexp(torch.where(torch.isinf(xt), torch.full_like(xt, -1e30), xt), 1, keepdim=True)
    else:
        lp = torch.nn.functional.logsigmoid(xt)
    lp = torch.gather(lp, 1, at)
    lp = torch.where(okt, lp, torch.full_like(lp, -1e30))
    if renorm:
        w = torch.where(okt, torch.softmax(lp, 1), torch.zeros_like(lp)) * scale
    else:
        w = torch.where(okt, torch.exp(lp), torch.zeros_like(lp)) * scale
    (w * gt).sum().backward()
    dx = torch.nan_to_num(xt.grad).numpy()
    wn = w.detach().numpy()
    # every gradient is a sum of terms no larger than these
    mag = np.zeros_like(x)
    share = (np.abs(wn) * np.abs(g)).sum(1, keepdims=True)
    for j in range(ids.shape[1]):
        add = np.where(ok[:, j], np.abs(wn[:, j]) * np.abs(g[:, j]), 0.0)
        if renorm:
            add = add + np.where(ok[:, j], np.abs(wn[:, j]) * share[:, 0] / abs(scale), 0.0)
        np.add.at(mag, (np.arange(x.shape[0]), np.where(ok[:, j], ids[:, j], 0)), add)
    if scores == "softmax" and not renorm:
        with np.errstate(over="ignore"):
            p = torch.softmax(torch.where(torch.isinf(xt), torch.full_like(xt, -1e30), xt), 1).detach().numpy()
        mag += p * share
    return dx, mag


TOP = {"e4m3": 448.0, "e5m2": 57344.0}


def fp8_values(v, fmt):
    """the 8-bit floats nearest to v (float64), ties to even, |v| <= top; NaN and (e4m3) infinities are NaN"""
    digits, least = (3, -6) if fmt == "e4m3" else (2, -14)
    a = np.abs(np.where(np.isfinite(v), v, 0.0))
    m, e = np.frexp(a)                              # a = m 2^e, m in [0.5, 1)
    step = np.exp2(np.maximum(e - 1, least) - digits)
    q = np.where(np.isfinite(v), np.round(np.where(np.isfinite(v), v, 0.0) / step) * step, v)
    if fmt == "e4m3":
        q = np.where(np.isinf(v), np.nan, q)
    return q


def fp8_exponent(top, fmt):
    """smallest e >= -110 with top <= TOP 2^e; 0 for top = 0"""
    e = -110
    if top == 0.0:
        return 0
    while top > TOP[fmt] * 2.0 ** e:
        e += 1
    return e


def fp8_blocks(x, fmt, rows, cols):
    """x (float64 numpy, 2-D) in blocks of rows x cols: (values, exponent of each block)"""
    R, C = x.shape
    out = np.zeros_like(x)
    es = np.zeros((-(-R // rows), -(-C // cols)), dtype=int)
    for i in range(es.shape[0]):
        for j in range(es.shape[1]):
            sl = (slice(i * rows, (i + 1) * rows), slice(j * cols, (j + 1) * cols))
            b = x[sl]
            f = b[np.isfinite(b)]
            e = fp8_exponent(np.abs(f).max() if f.size else 0.0, fmt)
            es[i, j] = e
            out[sl] = fp8_values(b / 2.0 ** e, fmt) * 2.0 ** e
    return out, es


def plan(ids, E):
    """(pair by row, expert by row, pos) of the stable order"""
    flat = ids.reshape(-1)
    ok = np.flatnonzero((flat >= 0) & (flat < E))
    pair = ok[np.argsort(flat[ok], kind="stable")]
    pos = np.full(flat.size, -1)
    pos[pair] = np.arange(pair.size)
    return pair, flat[pair], pos.reshape(ids.shape)


def wild(shape, seed, blockwise=True):
    """normal numbers whose magnitude changes from block to block, so that a wrong scale shows"""
    r = np.random.RandomState(seed)
    x = r.randn(*shape)
    if blockwise:
        R, C = shape[-2:]
        f = np.exp2(r.randint(-9, 10, (-(-R // 16), -(-C // 128)))).repeat(16, 0).repeat(128, 1)[:R, :C]
        x = x * f
    return x
