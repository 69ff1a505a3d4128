"""
Row-wise MLP blocks (pygho_amd/rowops.py) against their formulas in 64 bits on the same inputs.

Tolerances.  An output is the f32 result rounded once: half a step of its type (bf16 2^-8, f16 2^-11, f32 2^-24, relative to the value) plus
the f32 error of the steps before.  That part is bounded by (number of roundings on the longest chain) * 2^-24 * (the sum of the absolute
values that enter): the chains here are at most 64 lane-group additions + 32 serial ones + a handful per element, CHAIN = 128 covers them;
the hardware exp2 and reciprocal of the 16-bit types add a few 2^-22, covered by the same factor.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
CHAIN = 128 * 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
ACTS = ["none", "relu", "silu", "elu"]


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.device("cuda:0")


def act64(u, act):
    """(act(u), act'(u)) in 64 bits"""
    if act == "none":
        return u, torch.ones_like(u)
    if act == "relu":
        return torch.relu(u), (u > 0).double()
    if act == "silu":
        s = torch.sigmoid(u)
        return u * s, s * (1 + u * (1 - s))
    e = torch.expm1(torch.clamp(u, max=0.0))
    return torch.clamp(u, min=0.0) + e, torch.where(u > 0, torch.ones_like(u), e + 1)


def close(got, want, tol, what):
    err = (got.double() - want).abs()
    bad = ~(err <= tol) & ~(torch.isnan(got.double()) & torch.isnan(want)) & ~(got.double() == want)
    if bool(bad.any()):
        i = int(torch.where(bad.flatten(), (err / tol.clamp_min(1e-300)).flatten().nan_to_num(1e30), torch.zeros_like(err.flatten())).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, worst at {i}: got {got.flatten()[i].item()!r}, want "
                             f"{want.flatten()[i].item()!r}, tolerance {tol.flatten()[i].item():.3e}")


def grid_values(gen, shape, dev, scale, step=1.0 / 64):
    """random multiples of `step`: exactly representable in 16 bits, so that every dtype sees the same numbers"""
    return torch.randn(shape, generator=gen, device=dev).mul_(scale / step).round_().clamp_(-255, 255).mul_(step)


# ---- layer norm ---------------------------------------------------------------------------------------------------------------------
def ln_reference(x, w, b, eps, act, r, gy):
    """outputs, gradients and the absolute sums their tolerances count, in 64 bits"""
    x, gy = x.double(), gy.double()
    c = x.shape[1]
    g = torch.ones(c, dtype=torch.float64, device=x.device) if w is None else w.double()
    h = torch.zeros(c, dtype=torch.float64, device=x.device) if b is None else b.double()
    mean = x.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    xh = (x - mean) * rstd
    u = xh * g + h
    a, slope = act64(u, act)
    y = a if r is None else a + r.double()
    du = gy * slope
    e = du * g
    gx = rstd * (e - e.mean(1, keepdim=True) - xh * (e * xh).mean(1, keepdim=True))
    # what an error of one unit in the f32 chain may move: x and the mean scaled by rstd in xh, from there through g into u
    ax = (x.abs().amax(1, keepdim=True) + mean.abs()) * rstd + xh.abs()
    au = ax * g.abs() + h.abs()
    ay = au + a.abs() + (0 if r is None else r.double().abs())
    ae = gy.abs() * (1 + au) * g.abs()              # |act''| <= 1: an error of u moves du by at most that
    agx = rstd * (ae + ae.mean(1, keepdim=True) + (xh.abs() + ax) * (ae * (1 + ax)).mean(1, keepdim=True))
    gg, gh = (du * xh).sum(0), du.sum(0)
    agg, agh = (gy.abs() * (1 + au) * (1 + ax)).sum(0), (gy.abs() * (1 + au)).sum(0)
    return (y, ay), (gx, agx), (gg, agg), (gh, agh)


def ln_check(x, w, b, eps, act, r, gy, what):
    from pygho_amd import _ops
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (x, w, b, r)]
    y = _ops.layer_norm_act(leaves[0], leaves[1], leaves[2], eps, act, residual=leaves[3])
    c = x.shape[-1]
    want = ln_reference(x.reshape(-1, c), w, b, eps, act, None if r is None else r.reshape(-1, c), gy.reshape(-1, c))
    assert y.shape == x.shape and y.dtype == x.dtype
    close(y.reshape(-1, c), want[0][0], want[0][0].abs() * HALF[x.dtype] + CHAIN * want[0][1], what + " y")
    ask = [t for t in leaves if t is not None]
    grads = dict(zip([id(t) for t in ask], torch.autograd.grad(y, ask, gy)))
    gx = grads[id(leaves[0])]
    close(gx.reshape(-1, c), want[1][0], want[1][0].abs() * HALF[x.dtype] + CHAIN * want[1][1], what + " gx")
    for t, (g, a), name in ((leaves[1], want[2], "gw"), (leaves[2], want[3], "gb")):
        if t is not None:
            assert grads[id(t)].dtype == t.dtype and grads[id(t)].shape == t.shape
            close(grads[id(t)], g, g.abs() * HALF[t.dtype] + CHAIN * a, what + " " + name)
    if r is not None:
        assert torch.equal(grads[id(leaves[3])], gy)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,c,act", [(1, 1, "none"), (5, 2, "silu"), (63, 3, "elu"), (257, 8, "relu"), (130, 31, "silu"), (1000, 64, "silu"),
                                        (513, 100, "elu"), (2967, 128, "silu"), (77, 193, "relu"), (300, 256, "none"), (65, 257, "silu"),
                                        (129, 512, "elu"), (40, 1000, "silu"), (33, 1024, "relu"), (9, 1025, "silu"), (17, 2048, "elu"),
                                        (6, 2056, "silu"), (3, 5001, "none"), (20011, 32, "silu")])
def test_layer_norm_act(dev, dtype, rows, c, act):
    gen = torch.Generator(device=dev)
    gen.manual_seed(rows * 131 + c)
    x = grid_values(gen, (rows, c), dev, 1.0).add_(0.5).to(dtype)
    w = grid_values(gen, (c,), dev, 0.3).add_(1.0).to(dtype)
    b = grid_values(gen, (c,), dev, 0.3).to(dtype)
    r = grid_values(gen, (rows, c), dev, 1.0).to(dtype)
    gy = grid_values(gen, (rows, c), dev, 1.0).to(dtype)
    if act == "relu":
        # relu's slope jumps at 0: u is kept away from it (64 f32 steps of its own terms), where every correct sum agrees
        x64 = x.double()
        xh = (x64 - x64.mean(1, keepdim=True)) / torch.sqrt(x64.var(1, unbiased=False, keepdim=True) + 1e-5)
        u = xh * w.double() + b.double()
        gy = torch.where(u.abs() < 2.0 ** -16 * (1 + xh.abs() * w.double().abs() * 4), torch.zeros_like(gy), gy)
    print(f"layer_norm_act {rows} x {c} {act} {dtype}", flush=True)
    ln_check(x, w, b, 1e-5, act, r, gy, f"{rows}x{c} {act}")
    ln_check(x, None, None, 1e-3, act if act != "relu" else "silu", None, gy, f"{rows}x{c} plain {act}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_layer_norm_act_f32_parameters(dev, dtype):
    """master weights in f32 under 16-bit rows: gradients come back in f32"""
    gen = torch.Generator(device=dev)
    gen.manual_seed(3)
    for c in (128, 97):
        x, gy = (grid_values(gen, (700, c), dev, 1.0).to(dtype) for _ in range(2))
        ln_check(x, torch.randn(c, generator=gen, device=dev), torch.randn(c, generator=gen, device=dev), 1e-5, "silu", None, gy, f"f32 params {c}")
        ln_check(x, torch.randn(c, generator=gen, device=dev), grid_values(gen, (c,), dev, 1.0).to(dtype), 1e-5, "silu", None, gy, f"mixed {c}")


@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_norm_act_strides_and_dims(dev, dtype):
    gen = torch.Generator(device=dev)
    gen.manual_seed(4)
    big = grid_values(gen, (301, 300), dev, 1.0).to(dtype)
    w, b = (grid_values(gen, (128,), dev, 1.0).to(dtype) for _ in range(2))
    gy = grid_values(gen, (301, 300), dev, 1.0).to(dtype)
    for off in (0, 8, 1, 172):                                    # column slices: row stride 300, aligned and unaligned starts
        ln_check(big[:, off:off + 128], w, b, 1e-5, "silu", big[:, 100:228], gy[:, off:off + 128], f"slice {off}")
    ln_check(big[::3, :128], w, b, 1e-5, "elu", None, gy[::3, :128], "every third row")
    ln_check(big[:128].t(), w, b, 1e-5, "silu", None, gy[:128].t(), "transposed")
    ln_check(big[:1, :128].expand(50, 128), w, b, 1e-5, "silu", None, gy[:50, :128], "one row expanded")
    x4 = grid_values(gen, (3, 5, 7, 128), dev, 1.0).to(dtype)
    ln_check(x4, w, b, 1e-5, "silu", x4.flip(0), x4 * 0.5, "four dims")
    ln_check(x4.transpose(0, 2), w, b, 1e-5, "silu", None, x4.transpose(0, 2), "permuted dims")
    ln_check(x4[0, 0, 0], w, b, 1e-5, "silu", None, x4[1, 1, 1], "one row, one dim")
    # a gradient that autograd hands over expanded (stride 0 everywhere)
    from pygho_amd import _ops
    x = big[:, :128].detach().requires_grad_(True)
    a, = torch.autograd.grad(_ops.layer_norm_act(x, w, b, act="silu").sum(), x)
    c, = torch.autograd.grad(_ops.layer_norm_act(x, w, b, act="silu"), x, torch.ones_like(big[:, :128]).contiguous())
    assert torch.equal(a, c)


def test_layer_norm_act_hard_rows(dev):
    """constant rows (variance 0), a mean far from zero, tiny and huge rows, infinities and NaN: only the rows that hold them are touched"""
    from pygho_amd import _ops
    gen = torch.Generator(device=dev)
    gen.manual_seed(5)
    x = torch.randn(40, 128, generator=gen, device=dev)
    x[0] = 3.25
    x[1] = 0.0
    x[2] = x[2] * 2.0 ** -60
    x[3] = x[3] * 1e15
    x[4] = x[4] + 1000.0
    w, b, gy = torch.randn(128, generator=gen, device=dev), torch.randn(128, generator=gen, device=dev), torch.randn(40, 128, generator=gen, device=dev)
    ln_check(x, w, b, 1e-5, "silu", None, gy, "hard rows")
    for act in ACTS:
        clean = _ops.layer_norm_act(x, w, b, act=act)
        y = x.clone()
        y[7, 5], y[9, 0], y[11, 127] = float("inf"), float("nan"), float("-inf")
        out = _ops.layer_norm_act(y, w, b, act=act)
        keep = torch.ones(40, dtype=torch.bool, device=dev)
        keep[[7, 9, 11]] = False
        assert torch.equal(out[keep], clean[keep]) and torch.isnan(out[~keep]).any(1).all()
        gx, = torch.autograd.grad(_ops.layer_norm_act(y.requires_grad_(True), w, b, act=act), y, gy)
        want, = torch.autograd.grad(_ops.layer_norm_act(x.requires_grad_(True), w, b, act=act), x, gy)
        assert torch.equal(gx[keep], want[keep])
        x = x.detach()
    # eps = 0 on a row with a variance
    ln_check(x[5:], w, b, 0.0, "none", None, gy[5:], "eps 0")


def test_layer_norm_act_no_rows(dev):
    from pygho_amd import _ops
    for shape in ((0, 128), (3, 0, 64)):
        x = torch.zeros(shape, device=dev, requires_grad=True)
        w, b = torch.ones(shape[-1], device=dev, requires_grad=True), torch.zeros(shape[-1], device=dev, requires_grad=True)
        y = _ops.layer_norm_act(x, w, b, act="silu", residual=x)
        gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.zeros_like(y))
        assert y.shape == shape and gx.shape == shape and not gw.any() and not gb.any()


def test_layer_norm_act_gradients_against_differences(dev):
    """directional derivatives of <gy, y>: the kernel's gradients against central differences of the kernel's own f32 forward.  Step 2^-7: the
    difference is off by the third derivative's h^2 / 6 ~ 1e-5 of the gradient's scale and by 2^-24 * sqrt(n) |gy y| / h ~ 1e-4 of it"""
    from pygho_amd import _ops
    gen = torch.Generator(device=dev)
    gen.manual_seed(6)
    for act in ("none", "silu", "elu"):
        t = [torch.randn(50, 96, generator=gen, device=dev), torch.rand(96, generator=gen, device=dev) + 0.5, torch.randn(96, generator=gen, device=dev),
             torch.randn(50, 96, generator=gen, device=dev)]
        gy = torch.randn(50, 96, generator=gen, device=dev)
        leaves = [v.clone().requires_grad_(True) for v in t]
        grads = torch.autograd.grad(_ops.layer_norm_act(leaves[0], leaves[1], leaves[2], 1e-5, act, residual=leaves[3]), leaves, gy)
        for k in range(4):
            d = torch.randn(t[k].shape, generator=gen, device=dev)
            vals = []
            for s in (2.0 ** -7, -2.0 ** -7):
                a = [v + s * d if i == k else v for i, v in enumerate(t)]
                vals.append(float((_ops.layer_norm_act(a[0], a[1], a[2], 1e-5, act, residual=a[3]).double() * gy.double()).sum()))
            diff = (vals[0] - vals[1]) / 2.0 ** -6
            want = float((grads[k].double() * d.double()).sum())
            assert abs(diff - want) < 2e-3 * float(grads[k].double().norm() * d.double().norm()) / math.sqrt(d.numel()) + 2e-2, (act, k, diff, want)


def test_layer_norm_act_rows_counted_on_the_device(dev):
    """inside a batch slot (a capacity of rows, the true count on the device) the gradients are the bits of the exactly sized call, whatever
    the rows behind the count hold, and the rows of gx behind it stay as they were"""
    from pygho_amd import _ops
    gen = torch.Generator(device=dev)
    gen.manual_seed(7)
    for dtype in DTYPES:
        for c in (128, 100):
            w, b = (torch.randn(c, generator=gen, device=dev).to(dtype).requires_grad_(True) for _ in range(2))
            for true, cap in ((0, 64), (1, 50), (700, 1000), (1000, 1001), (5000, 40000), (33000, 40000)):
                x, gy = (torch.randn(cap, c, generator=gen, device=dev).to(dtype) for _ in range(2))
                x[true:] = float("nan")
                gy[true:] = float("inf")
                xe = x[:true].clone().requires_grad_(True)
                want = torch.autograd.grad(_ops.layer_norm_act(xe, w, b, act="silu"), (xe, w, b), gy[:true].clone())
                xc = x.requires_grad_(True)
                with _ops.row_families({cap: torch.tensor([true], dtype=torch.int32, device=dev)}):
                    y = _ops.layer_norm_act(xc, w, b, act="silu")
                    got = torch.autograd.grad(y, (xc, w, b), gy)
                assert torch.equal(got[0][:true], want[0]) and torch.equal(got[1], want[1]) and torch.equal(got[2], want[2]), (dtype, c, true, cap)


def test_layer_norm_act_repeats_and_streams(dev):
    """the same bits every time, from another stream as well"""
    from pygho_amd import _ops
    x = torch.randn(30011, 128, device=dev).bfloat16().requires_grad_(True)
    w, b = torch.randn(128, device=dev, requires_grad=True), torch.randn(128, device=dev, requires_grad=True)
    gy = torch.randn(30011, 128, device=dev).bfloat16()

    def once():
        y = _ops.layer_norm_act(x, w, b, act="silu", residual=x)
        return (y.detach(),) + torch.autograd.grad(y, (x, w, b), gy)
    first = once()
    for _ in range(3):
        assert all(torch.equal(a, b2) for a, b2 in zip(first, once()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = once()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b2) for a, b2 in zip(first, second))


def test_layer_norm_act_refusals(dev):
    from pygho_amd import _ops
    x = torch.randn(4, 8, device=dev)
    one = torch.ones(8, device=dev)
    for kw, exc in ((dict(x=x, act="gelu"), ValueError), (dict(x=x.double()), TypeError), (dict(x=x.long()), TypeError),
                    (dict(x=x, weight=one[:7]), ValueError), (dict(x=x, bias=one.double()), TypeError), (dict(x=x, residual=x[:3]), ValueError),
                    (dict(x=x, residual=x.half()), TypeError), (dict(x=x, eps=-1.0), ValueError), (dict(x=x, eps=float("nan")), ValueError),
                    (dict(x=x.reshape(-1)[0]), ValueError), (dict(x=x[:, :0]), ValueError), (dict(x=x, weight=one.cpu()), RuntimeError),
                    (dict(x=x.cpu()), RuntimeError)):
        with pytest.raises(exc):
            _ops.layer_norm_act(**kw)
    # second derivatives are refused, not wrong
    x = x.requires_grad_(True)
    g, = torch.autograd.grad(_ops.layer_norm_act(x, one, one, act="silu").square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)
