"""Cases for the mixture-of-experts operators: routing, expert products, combination, MXFP4.

Each case is one operator as a layer with experts calls it.  ``run`` computes it in plain
32-bit torch operations, or with this package's kernels where ``own`` is true; ``exact``
computes it in 64 bits from the definition.  Notation: T tokens, E experts, k experts per
token, R = T*k rows sorted by expert, K the width of the inputs, N that of the outputs.
"""

import math

import torch

own = False

LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)  # magnitudes of a 4-bit E2M1 code
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # One decode token through a router of 64 experts: launch latency.
        dict(name="route_token", op="route", T=1, E=64, k=8, dtype="bf16", renorm=True, mask=0.0, train=False),
        # A long prefill batch with 256 experts, masked experts and padding rows, and the
        # gradient of the logits.
        dict(name="route_train", op="route", T=8192, E=256, k=8, dtype="f32", renorm=False, mask=0.02, train=True),
        # A decode batch summed over its experts' rows.
        dict(name="combine_decode", op="combine", T=64, E=64, k=8, N=2048, dtype="bf16", skew=0.5, drop=0.0, train=False),
        # A training batch: the sum, and the gradients of the rows and of the weights.
        dict(name="combine_train", op="combine", T=8192, E=8, k=2, N=4096, dtype="bf16", skew=0.5, drop=0.01, train=True),
        # One decode token through its eight of 64 narrow experts: eight groups of one row.
        dict(name="experts_token", op="experts", T=1, E=64, k=8, K=2048, N=2048, dtype="bf16", skew=0.5, drop=0.0, train=False),
        # A chunk of mixed requests on many narrow experts: ragged groups, empty ones, padding.
        dict(name="experts_ragged", op="experts", T=1003, E=64, k=6, K=2048, N=1416, dtype="f16", skew=1.0, drop=0.03, train=False),
        # A long prefill on eight wide experts (the gate projection of 4096 -> 14336 layers).
        dict(name="experts_prefill", op="experts", T=8192, E=8, k=2, K=4096, N=14336, dtype="bf16", skew=0.3, drop=0.0, train=False),
        # A training step: the product and both gradients.
        dict(name="experts_train", op="experts", T=4096, E=16, k=4, K=2048, N=4096, dtype="bf16", skew=0.5, drop=0.01, train=True),
        # Activations of a decode batch to 4 bits.
        dict(name="quantize_decode", op="quantize", T=64, K=4096, dtype="bf16"),
        # A gate/up weight of 2 x 14336 rows to 4 bits, once per loaded checkpoint.
        dict(name="quantize_weight", op="quantize", T=28672, K=4096, dtype="bf16"),
        # A decode batch on wide experts kept in 4 bits: the weights' bytes count.
        dict(name="mx_decode", op="mx", T=16, E=8, k=2, K=4096, N=14336, dtype="bf16", skew=0.3, drop=0.0),
        # The long prefill with 4-bit weights and activations.
        dict(name="mx_prefill", op="mx", T=8192, E=8, k=2, K=4096, N=14336, dtype="bf16", skew=0.3, drop=0.0),
    ]


def _log_int(rng, lo, hi, step=1):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return max(lo, min(hi, max(step, v // step * step)))


def draw(rng):
    op = rng.choice(("route", "combine", "experts", "experts", "quantize", "mx", "mx"))
    T = _log_int(rng, 1, 8192)
    E = rng.choice((4, 8, 16, 40, 64, 128, 256))
    k = rng.randint(1, min(8, E))
    dtype = rng.choice(("bf16", "f16"))
    if op == "route":
        return dict(op=op, T=T, E=E, k=k, dtype=rng.choice(("bf16", "f16", "f32")), renorm=rng.random() < 0.5,
                    mask=rng.choice((0.0, 0.02, 0.3)), train=rng.random() < 0.5)
    if op == "quantize":
        return dict(op=op, T=_log_int(rng, 1, 28672), K=_log_int(rng, 64, 4096, 32), dtype=rng.choice(("bf16", "f16", "f32")))
    step = 32 if op == "mx" else 8
    N, K = _log_int(rng, 64, 8192, 8), _log_int(rng, 64, 5120, step)
    skew, drop = rng.choice((0.0, 0.5, 1.0)), rng.choice((0.0, 0.03, 0.2))
    train = rng.random() < 0.4
    # No drawn case is above the largest listed one's products, nor its weights' bytes.
    while 2 * T * k * N * (K if op != "combine" else 1) * (3 if train and op == "experts" else 1) > 1.9e12:
        T //= 2
    while E * N * K > 8 * 14336 * 4096:
        E, k = E // 2, min(k, E // 2)
    if op == "combine":
        return dict(op=op, T=T, E=E, k=k, N=N, dtype=dtype, skew=skew, drop=drop, train=train)
    case = dict(op=op, T=T, E=E, k=k, K=K, N=N, dtype=dtype, skew=skew, drop=drop)
    return case if op == "mx" else dict(case, train=train)


# ------------------------------------------------------------------ inputs
def _activations(g, rows, width, dtype):
    """Normal values whose channels differ in size, as a norm layer's outputs do."""
    channel = (0.5 * torch.randn(width, generator=g, device="cuda")).exp()
    return (torch.randn(rows, width, generator=g, device="cuda") * channel).to(dtype)


def _routing(g, case):
    """Experts of each token (popularity falls as a power of the index), sorted into rows."""
    T, E, k = case["T"], case["E"], case["k"]
    bias = -case["skew"] * torch.log(torch.arange(1, E + 1, device="cuda", dtype=torch.float32))
    u = torch.rand(T, E, generator=g, device="cuda").clamp_(1e-9, 1 - 1e-7)
    experts = (bias - torch.log(-torch.log(u))).topk(k, dim=1).indices
    experts[torch.rand(T, generator=g, device="cuda") < case["drop"]] = E  # padding tokens: no expert
    weights = torch.softmax(torch.randn(T, k, generator=g, device="cuda"), dim=1)
    order = torch.argsort(experts.reshape(-1), stable=True)
    counts = torch.bincount(experts.reshape(-1), minlength=E + 1)[:E]
    offsets = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = counts.cumsum(0)
    live = torch.arange(T * k, device="cuda") < offsets[E]
    rows = torch.where(live, order // k, -1).to(torch.int32)
    positions = torch.full((T * k,), -1, dtype=torch.int32, device="cuda")
    positions[order] = torch.where(live, torch.arange(T * k, device="cuda"), -1).to(torch.int32)
    return dict(weights=weights, offsets=offsets, rows=rows, positions=positions.view(T, k), counts=counts.tolist())


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, s = DTYPES[case["dtype"]], dict(case=case)
    if case["op"] in ("quantize", "mx"):  # what a scale byte and a code stand for; exact, unlike exp2 on the device
        s["powers"] = torch.tensor([2.0**i for i in range(-127, 128)], device="cuda")
        s["levels"] = torch.tensor(LEVELS + tuple(-v for v in LEVELS), device="cuda")
    if case["op"] == "route":
        T, E = case["T"], case["E"]
        logits = 1.5 * torch.randn(T, E, generator=g, device="cuda") + 0.5 * torch.randn(E, generator=g, device="cuda")
        if case["mask"]:  # experts that may not be taken, and padding tokens with none
            logits[torch.rand(T, E, generator=g, device="cuda") < case["mask"]] = -math.inf
            logits[torch.rand(T, generator=g, device="cuda") < case["mask"]] = -math.inf
        s["logits"] = logits.to(dtype)
        s["grad"] = torch.randn(T, case["k"], generator=g, device="cuda")
        return s
    if case["op"] == "quantize":
        s["x"] = _activations(g, case["T"], case["K"], dtype)
        return s
    s.update(_routing(g, case))
    T, E, R, N = case["T"], case["E"], case["T"] * case["k"], case["N"]
    if case["op"] == "combine":
        s["y"] = torch.randn(R, N, generator=g, device="cuda").to(dtype)
        s["grad"] = torch.randn(T, N, generator=g, device="cuda").to(dtype)
        return s
    K = case["K"]
    s["x"] = _activations(g, T, K, dtype)
    if case["op"] == "mx":  # a checkpoint's 4-bit weights: two codes a byte, a power of two for 32 values
        s["codes"] = torch.randint(0, 256, (E, N, K // 2), generator=g, device="cuda", dtype=torch.uint8)
        exponent = torch.randint(-2, 2, (E, N, K // 32), generator=g, device="cuda") - round(math.log2(K) / 2) + 127
        s["scales"] = exponent.to(torch.uint8)
        return s
    s["w"] = (torch.randn(E, N, K, generator=g, device="cuda", dtype=torch.bfloat16) / math.sqrt(K)).to(dtype)
    s["grad"] = torch.randn(R, N, generator=g, device="cuda", dtype=torch.bfloat16).to(dtype)
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    return globals()["_own_" + s["case"]["op"] if own else "_plain_" + s["case"]["op"]](s)


def _own_route(s):
    from loraforge_b200.ops.experts import route_experts, route_experts_backward

    c = s["case"]
    r = route_experts(s["logits"], c["k"], renormalize=c["renorm"])
    out = dict(weights=r.weights, experts=r.experts, offsets=r.offsets, rows=r.rows, positions=r.positions)
    if c["train"]:
        out["grad_logits"] = route_experts_backward(s["logits"], r, s["grad"], renormalize=c["renorm"])
    return out


def _own_combine(s):
    from loraforge_b200.ops.experts import combine_experts, combine_experts_backward

    out = dict(out=combine_experts(s["y"], s["weights"], s["positions"]))
    if s["case"]["train"]:
        out["grad_y"], out["grad_weights"] = combine_experts_backward(s["grad"], s["y"], s["weights"], s["positions"])
    return out


def _own_experts(s):
    from loraforge_b200.ops.experts import expert_linear, expert_linear_backward

    out = dict(y=expert_linear(s["x"], s["w"], s["offsets"], rows=s["rows"]))
    if s["case"]["train"]:
        out["grad_x"], out["grad_w"] = expert_linear_backward(s["grad"], s["x"], s["w"], s["offsets"], rows=s["rows"])
    return out


def _own_quantize(s):
    from loraforge_b200.ops.mxfp4 import mxfp4_dequantize, mxfp4_quantize

    return mxfp4_dequantize(mxfp4_quantize(s["x"]), torch.bfloat16)  # the 4-bit values as what they stand for


def _own_mx(s):
    from loraforge_b200.ops.mxfp4 import MxTensor, expert_linear_mxfp4, mxfp4_quantize

    return expert_linear_mxfp4(mxfp4_quantize(s["x"]), MxTensor(s["codes"], s["scales"]), s["offsets"], rows=s["rows"],
                               dtype=DTYPES[s["case"]["dtype"]])


def _plain_route(s):
    """p = softmax(logits); the k largest logits, ties to the lowest index; an expert at -inf is never taken."""
    c, logits = s["case"], s["logits"].float()
    T, E, k = c["T"], c["E"], c["k"]
    top, experts = torch.sort(logits, dim=1, descending=True, stable=True)
    top, experts = top[:, :k], experts[:, :k]
    taken = top > -math.inf
    peak = torch.where(taken[:, :1], top[:, :1], 0.0)
    e = torch.where(taken, (top - peak).exp(), 0.0)
    every = (logits - peak).exp()
    total = (e if c["renorm"] else every).sum(1, keepdim=True)
    weights = torch.where(taken, e / total, 0.0)
    experts = torch.where(taken, experts, -1)
    flat = torch.where(taken, experts, E).reshape(-1)
    order = torch.argsort(flat, stable=True)
    offsets = torch.zeros(E + 1, dtype=torch.int32, device=flat.device)
    offsets[1:] = torch.zeros(E + 1, dtype=torch.int64, device=flat.device).index_add_(0, flat, torch.ones_like(flat))[:E].cumsum(0)
    place = torch.arange(T * k, device=flat.device)
    live = place < offsets[E]
    rows = torch.where(live, order // k, -1)
    positions = torch.empty_like(order).index_copy_(0, order, torch.where(live, place, -1))
    out = dict(weights=weights, experts=experts.to(torch.int32), offsets=offsets, rows=rows.to(torch.int32),
               positions=positions.view(T, k).to(torch.int32))
    if c["train"]:
        spread = torch.zeros(T, E, device=flat.device).scatter_add_(1, experts.clamp(min=0), torch.where(taken, s["grad"], 0.0))
        if c["renorm"]:
            p = torch.zeros(T, E, device=flat.device).scatter_add_(1, experts.clamp(min=0), weights)
        else:
            p = torch.where(taken[:, :1], every / total, 0.0)
        out["grad_logits"] = (p * (spread - (p * spread).sum(1, keepdim=True))).to(s["logits"].dtype)
    return out


def _plain_combine(s):
    """out[t] = sum_j weights[t, j] * y[positions[t, j]]; a position of -1 adds nothing."""
    live = (s["positions"] >= 0)[..., None]
    at = s["positions"].clamp(min=0).long()
    y = torch.where(live, s["y"].float()[at], 0.0)
    out = dict(out=(s["weights"][..., None] * y).sum(1).to(s["y"].dtype))
    if s["case"]["train"]:
        grad = s["grad"].float()[:, None]
        out["grad_weights"] = (grad * y).sum(2)
        grad_y = torch.zeros(y.shape[0] * y.shape[1] + 1, y.shape[2], device=y.device)  # the last row takes the dropped ones
        to = torch.where(live[..., 0], at, y.shape[0] * y.shape[1]).reshape(-1)
        grad_y[to] = (s["weights"][..., None] * grad).reshape(-1, y.shape[2])
        out["grad_y"] = grad_y[:-1].to(s["y"].dtype)
    return out


def _plain_experts(s):
    """y[r] = W_e x[rows[r]] for the rows r of expert e; rows of no expert are zero."""
    live = (s["rows"] >= 0)[:, None]
    x = torch.where(live, s["x"].float()[s["rows"].clamp(min=0).long()], 0.0)
    R, (E, N, K) = x.shape[0], s["w"].shape
    train = s["case"]["train"]
    y = torch.zeros(R, N, device=x.device)
    if train:
        grad = s["grad"].float()
        grad_x, grad_w = torch.zeros_like(x), torch.zeros(E, N, K, device=x.device)
    lo = 0
    for e, n in enumerate(s["counts"]):  # no elementary product takes ragged groups
        if n:
            w, part = s["w"][e].float(), slice(lo, lo + n)
            y[part] = x[part] @ w.T
            if train:
                grad_x[part] = grad[part] @ w
                grad_w[e] = grad[part].T @ x[part]
        lo += n
    out = dict(y=y.to(s["x"].dtype))
    if train:
        out["grad_x"], out["grad_w"] = grad_x.to(s["x"].dtype), grad_w.to(s["w"].dtype)
    return out


def _plain_round4(x, powers):
    """Blocks of 32: scale 2^(floor(log2 amax) - 2), values to the nearest E2M1 (ties to even), at most 6."""
    b = x.float().unflatten(-1, (-1, 32))
    exponent = (torch.frexp(b.abs().amax(-1, keepdim=True)).exponent - 3).clamp(min=-127)
    v = b * powers[127 - exponent.long()]
    a = v.abs()
    q = torch.where(a < 2, (2 * a).round() / 2, torch.where(a < 4, a.round(), 2 * (a / 2).round())).clamp(max=6.0)
    return (torch.where(v < 0, -q, q) * powers[127 + exponent.long()]).flatten(-2)


def _plain_quantize(s):
    return _plain_round4(s["x"], s["powers"]).to(torch.bfloat16)


def _plain_mx(s):
    """The experts' products of 4-bit activations and 4-bit weights."""
    live = (s["rows"] >= 0)[:, None]
    x = torch.where(live, _plain_round4(s["x"], s["powers"])[s["rows"].clamp(min=0).long()], 0.0)
    y = torch.zeros(x.shape[0], s["codes"].shape[1], device=x.device)
    lo = 0
    for e, n in enumerate(s["counts"]):  # no elementary product takes ragged groups
        if n:
            codes = s["codes"][e].int()
            w = s["levels"][torch.stack((codes & 15, codes >> 4), -1).flatten(-2)].unflatten(-1, (-1, 32))
            w = (w * s["powers"][s["scales"][e].long()][..., None]).flatten(-2)
            y[lo : lo + n] = x[lo : lo + n] @ w.T
        lo += n
    return y.to(DTYPES[s["case"]["dtype"]])


# ------------------------------------------------------------------ bytes and operations
def work(case):
    op, T = case["op"], case["T"]
    size = 4 if case["dtype"] == "f32" else 2
    if op == "quantize":  # to 4.25 bits a value, and back to 16
        n = T * case["K"]
        return dict(bytes=n * (size + 2) + 2 * (n // 2 + n // 32), flops=4 * n)
    E, k = case["E"], case["k"]
    R = T * k
    if op == "route":
        out = R * 16 + 4 * E
        back = T * E * 2 * size + R * 12 if case["train"] else 0
        return dict(bytes=T * E * size + out + back, flops=T * E * (4 if not case["train"] else 10))
    N, live = case["N"], 1 - case["drop"]
    rows = R * live
    if op == "combine":
        back = size * (T * N + rows * N + R * N) + R * 8 if case["train"] else 0
        return dict(bytes=size * (rows * N + T * N) + R * 8 + back, flops=2 * rows * N * (3 if case["train"] else 1))
    K = case["K"]
    touched = _touched(case)
    flops = 2.0 * rows * N * K
    tokens = min(T, rows)
    if op == "mx":
        return dict(bytes=touched * N * K * 17 / 32 + tokens * K * 2 + R * N * 2 + R * 4, flops=flops)
    data = touched * N * K * 2 + tokens * K * 2 + R * N * 2 + R * 4
    if case["train"]:  # W, grad and x again; grad_x and grad_w out
        data += touched * N * K * 2 + 2 * rows * N * 2 + tokens * K * 2 + R * K * 2 + E * N * K * 2
    return dict(bytes=data, flops=flops * (3 if case["train"] else 1))


def _touched(case):
    """Expected number of experts with a token (each token's k draws are distinct)."""
    E, k, T = case["E"], case["k"], max(1.0, case["T"] * (1 - case["drop"]))
    share = [(i + 1.0) ** -case["skew"] for i in range(E)]
    total = sum(share)
    return sum(1 - max(0.0, 1 - min(1.0, k * p / total)) ** T for p in share)


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return globals()["_exact_" + case["op"]](s)


def _exact_route(s):
    c, l = s["case"], s["logits"].double().cpu()
    T, E, k = c["T"], c["E"], c["k"]
    ids = torch.arange(E).expand(T, E)
    chosen = torch.zeros(T, E, dtype=torch.bool)
    weights, which = torch.zeros(T, k, dtype=torch.float64), torch.full((T, k), -1)
    seen = torch.isfinite(l)
    alive = seen.any(1)
    z = torch.where(seen, torch.exp(l - torch.where(seen, l, -1e300).amax(1, keepdim=True)), 0.0)
    for j in range(k):
        rest = torch.where(seen & ~chosen, l, -math.inf)
        best = rest.amax(1, keepdim=True)
        pick = torch.where((rest == best) & (best > -math.inf), ids, E).amin(1)
        ok = pick < E
        which[ok, j] = pick[ok]
        chosen[ok, pick[ok]] = True
        weights[ok, j] = z[ok, pick[ok]]
    norm = torch.where(alive, (z * chosen).sum(1) if c["renorm"] else z.sum(1), 1.0)[:, None]
    weights /= norm
    out = dict(weights=weights, experts=None, offsets=None, rows=None, positions=None)
    if c["train"]:
        g = torch.zeros(T, E, dtype=torch.float64)
        t, j = torch.nonzero(which >= 0, as_tuple=True)
        g[t, which[t, j]] = s["grad"].double().cpu()[t, j]
        p = (z * chosen if c["renorm"] else z) / norm
        out["grad_logits"] = p * g - p * (p * g).sum(1, keepdim=True)
    return out


def _exact_combine(s):
    y, w, at = s["y"].double(), s["weights"].double(), s["positions"].long()
    out = torch.zeros(at.shape[0], y.shape[1], dtype=torch.float64, device=y.device)
    grad_y, grad_w = torch.zeros_like(y), torch.zeros_like(w)
    grad = s["grad"].double()
    for j in range(at.shape[1]):
        t = torch.nonzero(at[:, j] >= 0)[:, 0]
        r = at[t, j]
        out[t] += w[t, j, None] * y[r]
        grad_y[r] = w[t, j, None] * grad[t]
        grad_w[t, j] = torch.einsum("tn,tn->t", grad[t], y[r])
    return dict(out=out, grad_y=grad_y, grad_weights=grad_w) if s["case"]["train"] else dict(out=out)


def _exact_experts(s):
    E, N, K = s["w"].shape
    R = s["rows"].numel()
    bounds = s["offsets"].tolist()
    f64 = dict(dtype=torch.float64, device=s["w"].device)
    y, grad_x, grad_w = torch.zeros(R, N, **f64), None, None
    if s["case"]["train"]:
        grad_x, grad_w = torch.zeros(R, K, **f64), torch.zeros(E, N, K, **f64)
    for e in range(E):
        a, b = bounds[e], bounds[e + 1]
        if a == b:
            continue
        x, w = s["x"][s["rows"][a:b].long()].double(), s["w"][e].double()
        y[a:b] = torch.einsum("rk,nk->rn", x, w)
        if grad_x is not None:
            d = s["grad"][a:b].double()
            grad_x[a:b] = torch.einsum("rn,nk->rk", d, w)
            grad_w[e] = torch.einsum("rn,rk->nk", d, x)
    return dict(y=y, grad_x=grad_x, grad_w=grad_w) if grad_x is not None else dict(y=y)


def _exact_round4(x):
    """The same rounding by the distance to each level; on a tie the level whose code is even."""
    b = x.double().reshape(*x.shape[:-1], -1, 32)
    powers = torch.tensor([math.ldexp(1.0, i) for i in range(-127, 129)], dtype=torch.float64, device=b.device)
    largest = torch.bucketize(b.abs().amax(-1, keepdim=True), powers, right=True) - 1  # the last power not above it
    scale = powers[(largest - 2).clamp(min=0)]
    a, best, code = (b / scale).abs(), torch.zeros_like(b), torch.zeros_like(b)
    for i, level in enumerate(LEVELS[1:], 1):
        nearer, tie = (a - level).abs() < (a - best).abs(), (a - level).abs() == (a - best).abs()
        move = nearer | (tie & (i % 2 == 0))
        best, code = torch.where(move, level, best), torch.where(move, float(i), code)
    return (torch.sign(b) * best * scale).reshape(x.shape)


def _exact_quantize(s):
    return _exact_round4(s["x"])


def _exact_mx(s):
    bounds, x = s["offsets"].tolist(), _exact_round4(s["x"])
    table = torch.tensor(LEVELS + tuple(-v for v in LEVELS), dtype=torch.float64, device=x.device)
    powers = torch.tensor([math.ldexp(1.0, i - 127) for i in range(255)], dtype=torch.float64, device=x.device)
    E, N, half = s["codes"].shape
    y = torch.zeros(s["rows"].numel(), N, dtype=torch.float64, device=x.device)
    for e in range(E):
        a, b = bounds[e], bounds[e + 1]
        if a == b:
            continue
        w = torch.empty(N, 2 * half, dtype=torch.float64, device=x.device)
        w[:, 0::2], w[:, 1::2] = table[(s["codes"][e] % 16).long()], table[(s["codes"][e] // 16).long()]
        w *= powers[s["scales"][e].long()].repeat_interleave(32, dim=1)
        y[a:b] = torch.einsum("rk,nk->rn", x[s["rows"][a:b].long()], w)
    return y
