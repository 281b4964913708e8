"""The routing, 8-bit product and experts' product operators as cases: plain torch forms and the framework's calls.

`own` False computes an operator from elementary torch operations, True calls the framework.  The formulas:

route    p = softmax(x) or 1 / (1 + exp(-x)) over E experts; the choice goes by x itself or, with a bias or groups, by
         c = p + bias; a group's score is the sum of its two largest c; the k best of the experts that stay are taken in
         descending order, ties to the lowest index; a logit of -inf is a masked expert, an empty place has id -1 and
         weight 0; w = p (over its sum with renorm) * scale.
linear   y = x W' with x in blocks of 1 x 128 and W in blocks of 128 x 128 of 8-bit floats, each block scaled by the
         smallest power of two that brings it inside the format; dx = dy W, dW = dy' x with blocks of 128 rows.
experts  out_t = sum_j w_tj W_{e_tj} x_t on the same 8-bit products.
"""
import torch

own = False

DT = {"f64": torch.float64, "f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BLOCK = 128


# ---------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one token of a generation step through a router of 64 experts: launch latency
        {"name": "route_token", "op": "route", "T": 1, "E": 64, "k": 4, "scores": "softmax", "bias": False, "groups": 1,
         "group_k": 1, "renorm": True, "scale": 1.0, "dtype": "f32", "masked": False},
        # a long prompt's tokens, balance bias and groups, some experts masked and some rows padding
        {"name": "route_prompt", "op": "route", "T": 16384, "E": 256, "k": 8, "scores": "sigmoid", "bias": True,
         "groups": 8, "group_k": 4, "renorm": True, "scale": 2.5, "dtype": "f32", "masked": True},
        # the 20 best of a UBM's 512 components per frame, from the float64 log-probabilities of `logprob`
        {"name": "route_components", "op": "route", "T": 50001, "E": 512, "k": 20, "scores": "softmax", "bias": False,
         "groups": 1, "group_k": 1, "renorm": True, "scale": 1.0, "dtype": "f64", "masked": False},
        # a training step's router, forward and backward
        {"name": "route_train", "op": "route_train", "T": 32768, "E": 128, "k": 8, "scores": "softmax", "bias": True,
         "groups": 1, "group_k": 1, "renorm": True, "scale": 1.0, "dtype": "bf16", "masked": False},
        # one token through a linear layer: the weights' bytes
        {"name": "linear_token", "op": "linear", "M": 1, "N": 4096, "K": 4096, "dtype": "bf16"},
        # a small batch of generation steps
        {"name": "linear_batch", "op": "linear", "M": 61, "N": 8192, "K": 4096, "dtype": "bf16"},
        # whitened statistics of 1000 sessions (512 x 60) against a rank-400 loading matrix: few columns, long sums
        {"name": "linear_ragged", "op": "linear", "M": 1000, "N": 400, "K": 30720, "dtype": "f32"},
        # a prompt through a wide layer
        {"name": "linear_prompt", "op": "linear", "M": 8192, "N": 8192, "K": 8192, "dtype": "bf16"},
        # a training step of a layer: y, dx, dW from a batch that is no multiple of anything
        {"name": "linear_train", "op": "linear_train", "M": 8200, "N": 4096, "K": 4096, "dtype": "bf16", "grad": "e5m2"},
        # a few tokens of generation through 64 experts
        {"name": "experts_tokens", "op": "experts", "T": 8, "E": 64, "k": 4, "N": 2048, "K": 2048, "dtype": "bf16",
         "padded": False},
        # a padded prompt batch
        {"name": "experts_prompt", "op": "experts", "T": 8191, "E": 32, "k": 4, "N": 2048, "K": 4096, "dtype": "bf16",
         "padded": True},
        # a training step of the experts: out, dx, dW, dweights
        {"name": "experts_train", "op": "experts_train", "T": 8192, "E": 16, "k": 2, "N": 2048, "K": 2048,
         "dtype": "bf16", "grad": "e4m3", "padded": True},
    ]


def _size(rng, lo, hi):
    """log-uniform; one in three a multiple of 64, the others anything, odd ones among them"""
    v = int(round(lo * (hi / lo) ** rng.random()))
    if rng.random() < 0.34 and hi >= 64:
        v = min(hi, max(lo, (v + 63) // 64 * 64))
    return v


def draw(rng):
    op = rng.choice(["route", "route", "route_train", "linear", "linear", "linear_train", "experts", "experts",
                     "experts_train"])
    if op.startswith("route"):
        groups = rng.choice([1, 1, 4, 8])
        per = max(2, _size(rng, 8, 512) // groups)
        E = groups * per
        group_k = rng.randint(1, groups)
        k = rng.randint(2 if op.endswith("train") else 1, min(20, per * group_k))   # one weight of one has no gradient
        return {"op": op, "T": _size(rng, 1, 4000000 // E), "E": E, "k": k, "scores": rng.choice(["softmax", "sigmoid"]),
                "bias": rng.random() < 0.5, "groups": groups, "group_k": group_k, "renorm": rng.random() < 0.7,
                "scale": rng.choice([1.0, 2.5]), "dtype": rng.choice(["f32", "bf16", "f16"]),
                "masked": rng.random() < 0.5}
    if op.startswith("linear"):
        M, N, K = _size(rng, 1, 8192), _size(rng, 64, 8192), _size(rng, 64, 8192)
        case = {"op": op, "M": M, "N": N, "K": K, "dtype": rng.choice(["bf16", "bf16", "f16", "f32"])}
    else:
        E = _size(rng, 2, 64)
        T, N, K = _size(rng, 1, 8192), _size(rng, 64, 2048), _size(rng, 64, 2048)
        case = {"op": op, "T": T, "E": E, "k": rng.randint(1, min(E, 6)), "N": N, "K": K,
                "dtype": rng.choice(["bf16", "bf16", "f16"]), "padded": rng.random() < 0.5}
    if op.endswith("train"):
        case["grad"] = rng.choice(["e4m3", "e5m2"])
    return case


# ---------------------------------------------------------------------------------------------------- inputs
def _inputs(case, seed):
    """The tensors that a case's program holds, from the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + 17)
    dt = DT[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    if case["op"].startswith("route"):
        T, E, k = case["T"], case["E"], case["k"]
        spread = 12.0 if dt is torch.float64 else 1.5
        x = (normal(T, E) * spread + normal(1, E) - (100.0 if dt is torch.float64 else 0.0)).to(dt)
        if dt is torch.float64:     # 64-bit values are no widened 32-bit ones
            x += normal(T, E).double() * 1e-9
        if case["masked"]:          # experts that are switched off for a token, and padding rows
            x[uniform(T, E) < 0.05] = float("-inf")
            x[uniform(T) < 0.03] = float("-inf")
        s = {"logits": x}
        s["bias"] = normal(E) * 0.05 if case["bias"] else None
        if case["op"] == "route_train":
            s["dweights"] = normal(T, k) * 0.1
        return s
    K, N = case["K"], case["N"]
    rows = case["M"] if "M" in case else case["T"]
    # activations: a few strong channels, as behind a norm; weights of a layer's usual size
    x = (normal(rows, K) * (1.0 + 15.0 * (uniform(K) < 0.01))).to(dt)
    if "M" in case:
        s = {"x": x, "w": (normal(N, K) / K ** 0.5).to(dt)}
    else:
        E, T, k = case["E"], case["T"], case["k"]
        s = {"x": x, "w": torch.stack([(normal(N, K) / K ** 0.5).to(dt) for _ in range(E)])}
        liked = normal(1, E) * 0.5          # some experts are more popular than others
        scores = normal(T, E) + liked
        ids = torch.sort(scores, dim=1, descending=True, stable=True)[1][:, :k]
        w = torch.softmax(torch.gather(scores, 1, ids), dim=1)
        if case["padded"]:                  # padding tokens have no expert
            none = uniform(T) < 0.1
            ids = torch.where(none[:, None], torch.full_like(ids, -1), ids)
            w = torch.where(none[:, None], torch.zeros_like(w), w)
        s["ids"], s["weights"] = ids.int().contiguous(), w.contiguous()
    if case["op"].endswith("train"):
        s["dy"] = (normal(rows, N) * 1e-3).to(dt)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        import sidekit_amd
        s["engine"] = sidekit_amd.default_engine()
    if case["op"] in ("linear", "experts"):     # a serving program keeps its weights in their 8-bit form
        s["wq"] = s["engine"].fp8_tiles(s["w"]) if own else _tiles(s["w"], "e4m3")
        del s["w"]
    return s


# ---------------------------------------------------------------------------------------------------- plain forms
def _power(e):
    """2 ** e exactly, e an int32 tensor from -126 to 127 (a power function may be off in its last bits)"""
    return ((e.int() + 127) << 23).view(torch.float32)


def _quantized(x, fmt, dims):
    """x (float32) with each block, `dims` of x, in 8-bit floats with a power-of-two scale: the values they stand for"""
    m, e = torch.frexp(x.abs().amax(dim=dims, keepdim=True))
    e = e - (9 if fmt == "e4m3" else 16) + (m > 0.875).int()      # 448 = 0.875 * 2^9, 57344 = 0.875 * 2^16
    e = torch.where(m == 0, torch.zeros_like(e), e).clamp(min=-110)
    q = (x * _power(-e)).to(torch.float8_e4m3fn if fmt == "e4m3" else torch.float8_e5m2)
    return q.float() * _power(e)


def _blocked(x, dim):
    """x with zeros behind its last entry of `dim`, that axis split into blocks of 128"""
    dim %= x.dim()
    n = x.shape[dim]
    short = -n % BLOCK
    if short:
        x = torch.cat([x, x.new_zeros(*x.shape[:dim], short, *x.shape[dim + 1:])], dim)
    return x.reshape(*x.shape[:dim], (n + short) // BLOCK, BLOCK, *x.shape[dim + 1:])


def _rows(x, fmt):
    return _quantized(_blocked(x.float(), -1), fmt, (-1,)).flatten(-2)[..., :x.shape[-1]].contiguous()


def _columns(x, fmt):
    return _quantized(_blocked(x.float(), -2), fmt, (-2,)).flatten(-3, -2)[..., :x.shape[-2], :].contiguous()


def _tiles(w, fmt):
    b = _blocked(_blocked(w.float(), -2), -1)              # .., rows/128, 128, cols/128, 128
    b = _quantized(b, fmt, (-3, -1)).flatten(-2).flatten(-3, -2)
    return b[..., :w.shape[-2], :w.shape[-1]].contiguous()


def _route_plain(x, bias, c):
    T, E, k = c["T"], c["E"], c["k"]
    none = x == float("-inf")
    x = x.double()                                       # the order of near ties
    if c["scores"] == "softmax":
        top = x.amax(1, keepdim=True)
        p = torch.exp(x - torch.where(torch.isinf(top), torch.zeros_like(top), top))
        p = p / p.sum(1, keepdim=True).clamp(min=1e-300)
    else:
        p = 1 / (1 + torch.exp(-x))
    key = p + bias.double() if bias is not None else p if c["groups"] > 1 else x
    key = torch.where(none, torch.full_like(key, float("-inf")), key)
    if c["groups"] > 1:
        two = torch.sort(key.view(T, c["groups"], -1), dim=2, descending=True)[0][:, :, :2]
        score = torch.where(torch.isinf(two), torch.zeros_like(two), two).sum(2)
        score = torch.where(torch.isinf(two[:, :, 0]), two[:, :, 0], score)
        best = torch.sort(score, dim=1, descending=True, stable=True)[1][:, :c["group_k"]]
        stays = torch.zeros_like(score, dtype=torch.bool).scatter_(1, best, True)
        stays = stays[:, :, None].expand(T, c["groups"], E // c["groups"]).reshape(T, E)
        order = p if bias is None else key
        key = torch.where(stays & ~none, x if bias is None else order, torch.full_like(key, float("-inf")))
    key, ids = torch.sort(key, dim=1, descending=True, stable=True)
    key, ids = key[:, :k], ids[:, :k]
    there = key != float("-inf")
    w = torch.where(there, torch.gather(p, 1, ids), torch.zeros_like(key))
    if c["renorm"]:
        w = w / w.sum(1, keepdim=True).clamp(min=1e-300)
    return torch.where(there, ids, torch.full_like(ids, -1)).int(), (w * c["scale"]).float()


def _route_back_plain(x, ids, g, c):
    top = x.amax(1, keepdim=True)
    z = (x - torch.where(torch.isinf(top), torch.zeros_like(top), top)).float()
    if c["scores"] == "softmax":
        p = torch.exp(z)
        p = p / p.sum(1, keepdim=True).clamp(min=1e-30)
    else:
        p = 1 / (1 + torch.exp(-x.float()))
    there = ids >= 0
    at = ids.long().clamp(min=0)
    ps = torch.where(there, torch.gather(p, 1, at), torch.zeros_like(g))
    g = torch.where(there, g, torch.zeros_like(g))
    if c["renorm"]:
        total = ps.sum(1, keepdim=True).clamp(min=1e-30)
        g = (g - (g * ps).sum(1, keepdim=True) / total) / total
    u = torch.zeros_like(p).scatter_add_(1, at, torch.where(there, g * c["scale"], torch.zeros_like(g)))
    if c["scores"] == "softmax":
        dx = p * (u - (p * u).sum(1, keepdim=True))
    else:
        dx = p * (1 - p) * u
    return dx.to(x.dtype)


def _sorted(ids, E):
    """the (token, slot) pairs by expert, pairs without one last; their experts; the place of each in its expert"""
    flat = ids.flatten().long()
    expert = torch.where(flat < 0, torch.full_like(flat, E), flat)
    expert, order = torch.sort(expert, stable=True)
    count = torch.zeros(E + 1, dtype=torch.long, device=ids.device).scatter_add_(0, expert, torch.ones_like(expert))
    place = torch.arange(expert.numel(), device=ids.device) - (count.cumsum(0) - count)[expert]
    most = int(count[:E].max())
    n = int(count[:E].sum())
    return order[:n], expert[:n], place[:n], max(1, most)


def _experts_plain(x, ids, weights, wq, dtype):
    """(out, rows of every pair) with x and wq (E x N x K) the values of the 8-bit floats"""
    T, k = ids.shape
    E = wq.shape[0]
    order, expert, place, most = _sorted(ids, E)
    xp = x.new_zeros(E, most, x.shape[1])
    xp[expert, place] = x[order // k]
    y = torch.bmm(xp, wq.transpose(1, 2).contiguous())
    rows = x.new_zeros(T * k, wq.shape[1])
    rows[order] = y[expert, place]
    rows = rows.view(T, k, -1)
    return (rows * weights[:, :, None]).sum(1).to(dtype), rows


def _run_plain(s):
    c = s["case"]
    if c["op"].startswith("route"):
        ids, w = _route_plain(s["logits"], s["bias"], c)
        if c["op"] == "route":
            return ids, w
        return ids, w, _route_back_plain(s["logits"], ids, s["dweights"], c)
    x = s["x"]
    if c["op"] == "linear":
        return (_rows(x, "e4m3") @ s["wq"].t()).to(x.dtype)
    if c["op"] == "linear_train":
        wq = _tiles(s["w"], "e4m3")
        y = (_rows(x, "e4m3") @ wq.t()).to(x.dtype)
        dx = (_rows(s["dy"], c["grad"]) @ wq).to(x.dtype)
        dw = _columns(s["dy"], c["grad"]).t() @ _columns(x, "e4m3")
        return y, dx, dw
    ids, weights = s["ids"], s["weights"]
    if c["op"] == "experts":
        return _experts_plain(_rows(x, "e4m3"), ids, weights, s["wq"], x.dtype)[0]
    wq, dy = _tiles(s["w"], "e4m3"), s["dy"]
    out, rows = _experts_plain(_rows(x, "e4m3"), ids, weights, wq, x.dtype)
    dx = _experts_plain(_rows(dy, c["grad"]), ids, weights, wq.transpose(1, 2).contiguous(), x.dtype)[0]
    dweights = (rows * dy.float()[:, None, :]).sum(2)
    order, expert, place, most = _sorted(ids, c["E"])
    token = order // c["k"]
    xp = torch.zeros(c["E"], most, c["K"], device=x.device)
    dp = torch.zeros(c["E"], most, c["N"], device=x.device)
    xp[expert, place] = x[token].float()
    dp[expert, place] = dy[token].float() * weights.flatten()[order][:, None]
    dw = torch.bmm(_columns(dp, c["grad"]).transpose(1, 2).contiguous(), _columns(xp, "e4m3"))
    return out, dx, dw, dweights


# ---------------------------------------------------------------------------------------------------- the framework
def _run_own(s):
    c, eng = s["case"], s["engine"]
    if c["op"].startswith("route"):
        ids, w = eng.route(s["logits"], c["k"], scores=c["scores"], bias=s["bias"], groups=c["groups"],
                           group_k=c["group_k"], renorm=c["renorm"], scale=c["scale"])
        if c["op"] == "route":
            return ids, w
        return ids, w, eng.route_backward(s["logits"], ids, s["dweights"], scores=c["scores"], renorm=c["renorm"],
                                          scale=c["scale"])
    x = s["x"]
    if c["op"] == "linear":
        return eng.gemm_fp8(x, s["wq"], dtype=x.dtype)
    if c["op"] == "linear_train":
        dy = s["dy"]
        wq, wt = eng.fp8_tiles(s["w"], transposed=True)
        y = eng.gemm_fp8(eng.fp8_rows(x), wq, dtype=x.dtype)
        dx = eng.gemm_fp8(eng.fp8_rows(dy, c["grad"]), wt, dtype=x.dtype)
        dw = eng.gemm_fp8(eng.fp8_columns(dy, c["grad"]), eng.fp8_columns(x), dtype=torch.float32)
        return y, dx, dw
    plan = eng.route_plan(s["ids"], c["E"])
    if c["op"] == "experts":
        rows = eng.gemm_fp8_experts(x, s["wq"], plan, dtype=x.dtype)
        return eng.route_combine(rows, s["weights"], plan, dtype=x.dtype)
    dy, weights = s["dy"], s["weights"]
    wq, wt = eng.fp8_tiles(s["w"], transposed=True)
    rows = eng.gemm_fp8_experts(eng.fp8_rows(x), wq, plan, dtype=torch.float32)
    out = eng.route_combine(rows, weights, plan, dtype=x.dtype)
    back = eng.gemm_fp8_experts(eng.fp8_rows(dy, c["grad"]), wt, plan, dtype=x.dtype)
    dx = eng.route_combine(back, weights, plan, dtype=x.dtype)
    dweights = eng.route_combine_backward(rows, dy, plan)
    dw = eng.gemm_fp8_experts_wgrad(eng.fp8_columns(dy, c["grad"], plan=plan, weights=weights),
                                    eng.fp8_columns(x, plan=plan), plan)
    return out, dx, dw, dweights


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---------------------------------------------------------------------------------------------------- what it takes
def work(case):
    size = {"f64": 8, "f32": 4, "bf16": 2, "f16": 2}[case["dtype"]]
    if case["op"].startswith("route"):
        T, E, k = case["T"], case["E"], case["k"]
        moved = T * E * size + T * k * 8
        if case["op"] == "route_train":     # the logits are read again behind the loss, the gradient is written
            moved += 2 * T * E * size + T * k * 8
        return {"bytes": moved, "flops": 8 * T * E}
    N, K = case["N"], case["K"]
    if "M" in case:
        M = case["M"]
        if case["op"] == "linear":
            return {"bytes": M * K * size + N * K + M * N * size, "flops": 2 * M * N * K}
        return {"bytes": (2 * M * K + N * K + 2 * M * N) * size + 4 * N * K, "flops": 6 * M * N * K}
    T, E, k = case["T"], case["E"], case["k"]
    met = min(E, T * k)
    if case["op"] == "experts":
        return {"bytes": T * K * size + met * N * K + T * N * size + T * k * 8, "flops": 2 * T * k * N * K}
    return {"bytes": (2 * T * K + E * N * K + 2 * T * N) * size + 4 * E * N * K + T * k * 12,
            "flops": 6 * T * k * N * K}


# ---------------------------------------------------------------------------------------------------- in 64 bits
def _exact_blocks(v, fmt):
    """the 8-bit floats' values of v (float64, blocks along the last axis), from the definition of the format"""
    digits, least, top = (3, -6, 448.0) if fmt == "e4m3" else (2, -14, 57344.0)
    big = v.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(torch.where(big > 0, big, torch.ones_like(big)) / top))
    for shift in (-1, 1):           # log2 may round at a power of two
        t = e + shift
        fits = big <= top * torch.exp2(t)
        e = torch.where(fits if shift < 0 else ~(big <= top * torch.exp2(e)), t, e)
    scale = torch.where(big > 0, torch.exp2(e.clamp(min=-110)), torch.ones_like(big))
    a = v / scale
    octave = torch.floor(torch.log2(a.abs().clamp(min=2.0 ** least)))
    octave = torch.where(torch.exp2(octave) > a.abs().clamp(min=2.0 ** least), octave - 1, octave)
    octave = torch.where(torch.exp2(octave + 1) <= a.abs(), octave + 1, octave)
    step = torch.exp2(octave - digits)
    return torch.round(a / step) * step * scale


def _exact_matrix(x, fmt, tile=False):
    """rows in blocks of 128 along the last axis, or tiles of 128 x 128"""
    r, c = x.shape
    rp, cp = (-r % BLOCK if tile else 0), -c % BLOCK
    v = torch.nn.functional.pad(x.double(), (0, cp, 0, rp))
    if tile:
        v = v.view((r + rp) // BLOCK, BLOCK, -1, BLOCK).transpose(1, 2).reshape(-1, BLOCK * BLOCK)
        v = _exact_blocks(v, fmt).view((r + rp) // BLOCK, -1, BLOCK, BLOCK).transpose(1, 2)
    else:
        v = _exact_blocks(v.view(r, -1, BLOCK), fmt)
    return v.reshape(r + rp, c + cp)[:r, :c]


def _exact_route(s, c):
    x, bias = s["logits"].double(), s["bias"]
    T, E, k, G = c["T"], c["E"], c["k"], c["groups"]
    none = torch.isneginf(x)
    if c["scores"] == "softmax":
        logp = torch.nan_to_num(torch.log_softmax(x, 1), nan=float("-inf"), neginf=float("-inf"))
    else:
        logp = torch.nn.functional.logsigmoid(x)
    p = torch.exp(logp)
    choice = x if bias is None else p + bias.double()
    choice = choice.masked_fill(none, float("-inf"))
    if G > 1:
        c2 = (p if bias is None else choice).masked_fill(none, float("-inf")).view(T, G, E // G)
        first, at = c2.max(2)
        second = c2.scatter(2, at[:, :, None], float("-inf")).amax(2)
        score = first + second.masked_fill(torch.isneginf(second), 0.0)
        for g in range(G):          # a group stays if fewer than group_k are better or equal and before it
            ahead = (score > score[:, g:g + 1]).sum(1) + (score[:, :g] == score[:, g:g + 1]).sum(1)
            choice[:, g * (E // G):(g + 1) * (E // G)].masked_fill_((ahead >= c["group_k"])[:, None], float("-inf"))
    ids, logw = [], []
    left = choice.clone()
    for _ in range(k):
        best = left.amax(1, keepdim=True)
        at = (left == best).int().argmax(1, keepdim=True)        # the lowest index of the largest
        empty = torch.isneginf(best)
        ids.append(torch.where(empty, torch.full_like(at, -1), at))
        logw.append(torch.gather(logp, 1, at).masked_fill(empty, float("-inf")))
        left.scatter_(1, at, float("-inf"))
    ids, logw = torch.cat(ids, 1), torch.cat(logw, 1)
    w = torch.nan_to_num(torch.softmax(logw, 1), nan=0.0) if c["renorm"] else torch.exp(logw)
    return ids, w * c["scale"], p


def exact(case, seed):
    s = _inputs(case, seed)
    c = case
    if c["op"].startswith("route"):
        ids, w, p = _exact_route(s, c)
        out = (ids.int(), w)
        if c["op"] == "route":
            return out
        there = ids >= 0
        g = s["dweights"].double() * there
        if c["renorm"]:             # w_j = scale * share_j: d share / d p through the quotient
            ps = torch.gather(p, 1, ids.clamp(min=0)) * there
            total = ps.sum(1, keepdim=True)
            total = torch.where(total > 0, total, torch.ones_like(total))
            g = g / total - (g * ps).sum(1, keepdim=True) / total ** 2
        dp = torch.zeros_like(p)
        dp.scatter_add_(1, ids.clamp(min=0), g * there * c["scale"])
        if c["scores"] == "softmax":
            dx = p * dp - p * (p * dp).sum(1, keepdim=True)
        else:
            dx = dp * p * torch.sigmoid(-s["logits"].double())
        return out + (dx,)
    x = s["x"]
    xq = _exact_matrix(x, "e4m3")
    if c["op"].startswith("linear"):
        wq = _exact_matrix(s["w"], "e4m3", tile=True)
        if c["op"] == "linear":
            return xq @ wq.t()
        dy = s["dy"]
        return (xq @ wq.t(), _exact_matrix(dy, c["grad"]) @ wq,
                _exact_matrix(dy.t(), c["grad"]) @ _exact_matrix(x.t(), "e4m3").t())
    T, E, k, N, K = c["T"], c["E"], c["k"], c["N"], c["K"]
    train = c["op"] == "experts_train"
    ids, weights = s["ids"].long(), s["weights"]
    out = torch.zeros(T, N, dtype=torch.float64, device=x.device)
    if train:
        dy = s["dy"]
        dyq = _exact_matrix(dy, c["grad"])
        dx = torch.zeros(T, K, dtype=torch.float64, device=x.device)
        dw = torch.zeros(E, N, K, dtype=torch.float64, device=x.device)
        dweights = torch.zeros(T, k, dtype=torch.float64, device=x.device)
    for e in range(E):
        token, slot = torch.nonzero(ids == e, as_tuple=True)     # in the order of token, slot
        if not token.numel():
            continue
        we = _exact_matrix(s["w"][e], "e4m3", tile=True)
        share = weights[token, slot]
        y = xq[token] @ we.t()
        out.index_add_(0, token, y * share.double()[:, None])
        if train:
            dx.index_add_(0, token, (dyq[token] @ we) * share.double()[:, None])
            dweights[token, slot] = (y * dy[token].double()).sum(1)
            # the weighted gradient of a pair is a float32 number before it is quantized
            part = (dy[token].float() * share[:, None]).double()
            dw[e] = _exact_matrix(part.t(), c["grad"]) @ _exact_matrix(x[token].t(), "e4m3").t()
    return (out, dx, dw, dweights) if train else out
