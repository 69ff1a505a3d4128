"""
What is measured of the row-wise block operators: the cases, their inputs, the operators in plain torch and the calls a program makes.

Three operators over (rows, width) activations, the pieces an MLP with LayerNorm (or without a norm) is made of:

    layer_norm_act    y = act(LayerNorm(x) * g + h) + r
    linear_act        y = act(x W^T + b) + r
    linear_norm_act   y = act(LayerNorm(x W^T + b) * g + h) + r

each as the forward pass alone (a prediction) or as the forward and the backward pass for a given output gradient (a training step).
Widths and row counts are those of this package's models: hidden sizes 64 .. 512, node-level rows (a few thousand), tuple-level rows
(10^5 .. 10^6), graph-level rows (the batch).
"""
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
EPS = 1e-5


def _case(op, train, rows, width_in, width_out, dtype, act, bias=True, residual=False, name=None):
    c = {"op": op, "train": train, "rows": rows, "in": width_in, "out": width_out, "dtype": dtype, "act": act, "bias": bias,
         "residual": residual}
    if name is not None:
        c["name"] = name
    return c


def listed():
    return [
        # the readout of a 128-graph batch: one row per graph, latency only
        _case("layer_norm_act", False, 128, 128, 128, "f32", "silu", name="norm graphs f32"),
        # node-level rows of a 1024-graph batch at a width that is no power of two, training in f32
        _case("layer_norm_act", True, 23719, 193, 193, "f32", "elu", name="norm nodes odd f32 train"),
        # a wide row (concatenated views), half precision, prediction
        _case("layer_norm_act", False, 40531, 1000, 1000, "f16", "relu", residual=True, name="norm wide f16"),
        # tuple-level rows of an 8192-graph batch: the largest norm of a training step
        _case("layer_norm_act", True, 1831936, 128, 128, "bf16", "silu", residual=True, name="norm tuples bf16 train"),
        # the prediction head of a 128-graph batch: 128 -> 1
        _case("linear_act", False, 128, 128, 1, "f32", "none", name="linear head f32"),
        # node-level Linear of a 128-graph batch: launches, not bandwidth
        _case("linear_act", True, 2967, 128, 128, "bf16", "silu", name="linear nodes bf16 train"),
        # an f32 model of odd widths
        _case("linear_act", True, 60217, 97, 65, "f32", "elu", name="linear odd f32 train"),
        # three concatenated tuple representations -> hidden, tuple-level rows of a 1024-graph batch, with the residual connection
        _case("linear_act", True, 228992, 384, 128, "bf16", "silu", residual=True, name="linear concat bf16 train"),
        # tuple-level rows of 3-tuple batches at hidden 256, prediction
        _case("linear_act", False, 2386620, 256, 256, "bf16", "relu", name="linear 3-tuples bf16"),
        # node-level block of a 128-graph batch, prediction in half precision
        _case("linear_norm_act", False, 2967, 128, 128, "f16", "silu", residual=True, name="block nodes f16"),
        # the block of every layer of a training step on an 8192-graph batch
        _case("linear_norm_act", True, 1831936, 128, 128, "bf16", "silu", residual=True, name="block tuples bf16 train"),
        # hidden 512: the matrix products bound it
        _case("linear_norm_act", True, 65536, 512, 512, "bf16", "silu", residual=True, name="block wide bf16 train"),
    ]


# no drawn case costs more than the largest listed ones: "linear 3-tuples bf16" in products, "block tuples bf16 train" in bytes
_MAX_BYTES = 1.4e9
_MAX_FLOPS = 1.2e11


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng):
    if rng.random() < 0.45:
        return rng.choice([32, 64, 96, 128, 192, 256, 320, 384, 512])
    return _log_int(rng, 1, 1024)


def draw(rng):
    op = rng.choice(["layer_norm_act", "linear_act", "linear_norm_act"])
    train = rng.random() < 0.6
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    w_in = _width(rng)
    w_out = w_in if op == "layer_norm_act" or rng.random() < 0.3 else _width(rng)
    if op != "linear_act":                  # a norm over one or two channels returns the bias or signs
        w_in, w_out = (max(w_in, 8), max(w_out, 8)) if op == "linear_norm_act" else (max(w_in, 8),) * 2
    # relu's derivative jumps at 0, where two correct sums may land on different sides: prediction only
    act = rng.choice(["silu", "silu", "elu", "none"] if train else ["silu", "relu", "elu", "none"])
    case = _case(op, train, 1, w_in, w_out, dtype, act, bias=rng.random() < 0.8, residual=rng.random() < 0.5)
    one = work(dict(case, rows=1 << 20))
    most = (1 << 20) * min(_MAX_BYTES / one["bytes"], _MAX_FLOPS / one["flops"])
    case["rows"] = _log_int(rng, 1, max(2, min(2400000, int(most))))
    return case


def _linear(case):
    return case["op"] != "layer_norm_act"


def _norm(case):
    return case["op"] != "linear_act"


def work(case):
    m, k, n = case["rows"], case["in"], case["out"]
    size = 4 if case["dtype"] == "f32" else 2
    elems = m * k + m * n + (m * n if case["residual"] else 0)          # x, y, the residual
    params = (k * n if _linear(case) else 0) + (n if _linear(case) and case["bias"] else 0) + (2 * n if _norm(case) else 0)
    flops = (2.0 * m * k * n if _linear(case) else 0.0) + m * n * ((8 if _norm(case) else 0) + 4)
    if case["train"]:
        elems += m * n + m * k                                          # the output gradient in, x's gradient out (the residual's is the output gradient)
        params *= 2
        flops = (6.0 * m * k * n if _linear(case) else 0.0) + m * n * ((22 if _norm(case) else 0) + 10)
    return {"bytes": float((elems + params) * size), "flops": float(flops)}


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    m, k, n = case["rows"], case["in"], case["out"]

    def normal(*shape, scale=1.0, shift=0.0):
        return torch.randn(*shape, generator=gen, device=dev).mul_(scale).add_(shift).to(dt)

    def uniform(*shape, bound):
        return torch.rand(*shape, generator=gen, device=dev).mul_(2 * bound).sub_(bound).to(dt)

    s = {"case": dict(case), "x": normal(m, k, shift=0.25)}
    if _linear(case):
        s["w"] = uniform(n, k, bound=1.0 / math.sqrt(k))
        s["b"] = uniform(n, bound=1.0 / math.sqrt(k)) if case["bias"] else None
    if _norm(case):
        s["g"] = normal(n, scale=0.2, shift=1.0)
        s["h"] = normal(n, scale=0.2)
    s["r"] = normal(m, n) if case["residual"] else None
    s["gy"] = normal(m, n) if case["train"] else None
    s["leaves"] = [t for t in (s["x"], s["r"], s.get("w"), s.get("b"), s.get("g"), s.get("h")) if t is not None]
    if case["train"]:
        for t in s["leaves"]:
            t.requires_grad_(True)
    return s


def run(state):
    case = state["case"]
    if own:
        return _run_own(state)
    with torch.no_grad():
        out = _run_plain(state)
    return out if case["train"] else out[0]


def _call_own(state):
    from pygho_amd import _ops
    case = state["case"]
    if case["op"] == "layer_norm_act":
        return _ops.layer_norm_act(state["x"], state["g"], state["h"], EPS, case["act"], residual=state["r"])
    if case["op"] == "linear_act":
        return _ops.linear_act(state["x"], state["w"], state["b"], case["act"], residual=state["r"])
    return _ops.linear_norm_act(state["x"], state["w"], state["b"], state["g"], state["h"], EPS, case["act"], residual=state["r"])


def _run_own(state):
    if not state["case"]["train"]:
        with torch.no_grad():
            return _call_own(state)
    y = _call_own(state)
    return (y.detach(),) + torch.autograd.grad(y, state["leaves"], state["gy"])


def _act(z, act):
    """(act(z), act'(z)) in z's own precision"""
    if act == "none":
        return z, None
    if act == "relu":
        on = (z > 0).to(z.dtype)
        return z * on, on
    if act == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return z * s, s * (1.0 + z * (1.0 - s))
    neg = torch.clamp(z, max=0.0)
    e = torch.expm1(neg)
    return torch.clamp(z, min=0.0) + e, torch.where(z > 0, torch.ones_like(z), e + 1.0)


def _run_plain(state):
    """the operator and its gradients from their formulas, every intermediate in 32 bits (sums over the rows of f32 data in 64)"""
    case = state["case"]
    dt = state["x"].dtype
    wide = torch.float64 if dt == torch.float32 else torch.float32
    f = {k: (state[k].detach().float() if state.get(k) is not None else None) for k in ("x", "w", "b", "g", "h", "r", "gy")}
    z = f["x"]
    if _linear(case):
        z = z @ f["w"].t()
        if f["b"] is not None:
            z = z + f["b"]
    if _norm(case):
        mean = z.mean(1, keepdim=True)
        cen = z - mean
        rstd = 1.0 / torch.sqrt((cen * cen).mean(1, keepdim=True) + EPS)
        xhat = cen * rstd
        u = xhat * f["g"] + f["h"]
    else:
        u = z
    y, slope = _act(u, case["act"])
    if f["r"] is not None:
        y = y + f["r"]
    y = y.to(dt)
    if not case["train"]:
        return (y,)
    du = f["gy"] if slope is None else f["gy"] * slope
    gg = gh = None
    if _norm(case):
        gg = (du * xhat).sum(0, dtype=wide)
        gh = du.sum(0, dtype=wide)
        dx = du * f["g"]
        dz = rstd * (dx - dx.mean(1, keepdim=True) - xhat * (dx * xhat).mean(1, keepdim=True))
    else:
        dz = du
    gw = gb = None
    if _linear(case):
        gx = dz @ f["w"]
        gw = dz.to(wide).t() @ f["x"].to(wide)
        if f["b"] is not None:
            gb = dz.sum(0, dtype=wide)
    else:
        gx = dz
    grads = [gx, f["gy"] if f["r"] is not None else None, gw, gb, gg, gh]
    return (y,) + tuple(g.to(dt) for g in grads if g is not None)


def exact(case, seed):
    """the definition in 64 bits; the gradients by differentiating it"""
    state = prepare(case, seed)
    d = {k: (state[k].detach().to(torch.float64) if state.get(k) is not None else None) for k in ("x", "w", "b", "g", "h", "r", "gy")}
    leaves = [d[k] for k in ("x", "r", "w", "b", "g", "h") if d[k] is not None]
    for t in leaves:
        t.requires_grad_(case["train"])
    del state
    with torch.set_grad_enabled(case["train"]):
        z = d["x"]
        if _linear(case):
            z = torch.matmul(z, d["w"].transpose(0, 1))
            z = z if d["b"] is None else z + d["b"]
        if _norm(case):
            var, mean = torch.var_mean(z, dim=1, keepdim=True, unbiased=False)
            z = (z - mean) * torch.rsqrt(var + EPS) * d["g"] + d["h"]
        act = case["act"]
        if act == "relu":
            z = torch.relu(z)
        elif act == "silu":
            z = z * torch.sigmoid(z)
        elif act == "elu":
            z = torch.where(z > 0, z, torch.expm1(torch.minimum(z, torch.zeros_like(z))))
        y = z if d["r"] is None else z + d["r"]
        if not case["train"]:
            return y
        return (y.detach(),) + torch.autograd.grad(y, leaves, d["gy"])
