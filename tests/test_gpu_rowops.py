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


# ---- linear maps --------------------------------------------------------------------------------------------------------------------
# exact products: small integers, so that every partial sum in f32 is exact in any order and the only rounding is the last one
SHAPES = [(1, 1, 1), (1, 128, 1), (2, 3, 5), (17, 8, 16), (63, 33, 17), (64, 64, 64), (65, 65, 65), (128, 128, 1), (129, 100, 130), (200, 97, 65),
          (257, 129, 193), (300, 384, 128), (511, 256, 256), (1000, 128, 128), (77, 1000, 40), (40, 40, 1000), (300, 512, 512), (2967, 64, 96),
          (40000, 32, 48)]


def integers(gen, shape, dev, most):
    return torch.randint(-most, most + 1, shape, generator=gen, device=dev)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_linear_act_exact_products(dev, dtype, m, k, n):
    from pygho_amd import _ops
    gen = torch.Generator(device=dev)
    gen.manual_seed(m * 7 + k * 3 + n)
    print(f"linear_act {m} x {k} -> {n} {dtype}", flush=True)
    x, w, b, r, gy = (integers(gen, s, dev, most).to(dtype) for s, most in (((m, k), 3), ((n, k), 2), ((n,), 9), ((m, n), 4), ((m, n), 2)))
    for act, res in (("none", None), ("relu", r)):
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b)] + ([] if res is None else [res.clone().requires_grad_(True)])
        y = _ops.linear_act(leaves[0], leaves[1], leaves[2], act, residual=leaves[3] if res is not None else None)
        z = x.double() @ w.double().t() + b.double()
        a = torch.relu(z) if act == "relu" else z
        want = a if res is None else a + res.double()
        assert y.dtype == dtype and torch.equal(y, want.to(dtype))
        dz = gy.double() * (z > 0).double() if act == "relu" else gy.double()
        grads = torch.autograd.grad(y, leaves, gy)
        assert torch.equal(grads[0], (dz @ w.double()).to(dtype))
        assert torch.equal(grads[1], (dz.t() @ x.double()).to(dtype))
        assert torch.equal(grads[2], dz.sum(0).to(dtype))
        if res is not None:
            assert torch.equal(grads[3], gy)


def block_reference(x, w, b, g, h, eps, act, r, gy, normed):
    """outputs and gradients in 64 bits with bounds of what one unit of the f32 chain (u) and one rounding of dz to its 16-bit type (hr, 0 for
    f32) may move in each: {name: (value, f32 bound in units of 2^-24, bound of the rounding of dz)}"""
    x, w, gy = x.double(), w.double(), gy.double()
    k, n = x.shape[1], w.shape[0]
    z = x @ w.t() + (0 if b is None else b.double())
    cz = (k + 64) * (x.abs() @ w.abs().t() + (0 if b is None else b.double().abs()))          # a sum of k products, any order
    if normed:
        gw = torch.ones(n, dtype=torch.float64, device=x.device) if g is None else g.double()
        hw = torch.zeros(n, dtype=torch.float64, device=x.device) if h is None else h.double()
        mean = z.mean(1, keepdim=True)
        rstd = 1.0 / torch.sqrt(((z - mean) ** 2).mean(1, keepdim=True) + eps)
        xh = (z - mean) * rstd
        u = xh * gw + hw
        # xh moves with z, the mean (as z on average) and rstd (relative error rstd * mean of |dz| of the row)
        cxh = rstd * (cz + cz.mean(1, keepdim=True)) + xh.abs() * (rstd * cz * 2).mean(1, keepdim=True) + 64 * (xh.abs() + rstd * (z.abs() + mean.abs()))
        cu = cxh * gw.abs() + 8 * (u.abs() + hw.abs())
    else:
        u, cu = z, cz
    a, slope = act64(u, act)
    y = a if r is None else a + r.double()
    cy = 1.1 * cu + 8 * (a.abs() + (0 if r is None else r.double().abs()))
    du = gy * slope
    cdu = gy.abs() * (cu + 16)                        # |act''| <= 1
    out = {"y": (y, cy, torch.zeros_like(y))}
    if normed:
        out["gg"] = ((du * xh).sum(0), (cdu * xh.abs() + du.abs() * cxh + 128 * (du * xh).abs()).sum(0), torch.zeros(n, dtype=torch.float64, device=x.device))
        out["gh"] = (du.sum(0), (cdu + 128 * du.abs()).sum(0), torch.zeros(n, dtype=torch.float64, device=x.device))
        e, ce = du * gw, cdu * gw.abs() + 8 * (du * gw).abs()
        k2 = (e * xh).mean(1, keepdim=True)
        dz = rstd * (e - e.mean(1, keepdim=True) - xh * k2)
        ck2 = (ce * xh.abs() + e.abs() * cxh + 64 * (e * xh).abs()).mean(1, keepdim=True)
        cdz = rstd * (ce + (ce + 64 * e.abs()).mean(1, keepdim=True) + cxh * k2.abs() + xh.abs() * ck2 + 16 * (e.abs() + (xh * k2).abs()))
        cdz = cdz + dz.abs() * (rstd * cz * 2).mean(1, keepdim=True)
    else:
        dz, cdz = du, cdu
    out["gx"] = (dz @ w, cdz @ w.abs() + (n + 64) * (dz.abs() @ w.abs()), dz.abs() @ w.abs())
    m = x.shape[0]
    rows = min(m, 1024) + 256                         # longest chain of the split sum over the rows
    out["gw"] = (dz.t() @ x, cdz.t() @ x.abs() + rows * (dz.abs().t() @ x.abs()), dz.abs().t() @ x.abs())
    out["gb"] = (dz.sum(0), cdz.sum(0) + rows * dz.abs().sum(0), dz.abs().sum(0))
    return out


def block_check(normed, x, w, b, g, h, eps, act, r, gy, what):
    from pygho_amd import _ops
    names = ("x", "w", "b", "g", "h", "r")
    leaf = {k: (None if v is None else v.detach().clone(memory_format=torch.preserve_format).requires_grad_(True))
            for k, v in zip(names, (x, w, b, g, h, r))}
    leaf["x"] = x.detach().requires_grad_(True)            # (keeps its strides)
    if normed:
        y = _ops.linear_norm_act(leaf["x"], leaf["w"], leaf["b"], leaf["g"], leaf["h"], eps, act, residual=leaf["r"])
    else:
        y = _ops.linear_act(leaf["x"], leaf["w"], leaf["b"], act, residual=leaf["r"])
    k, n = w.shape[1], w.shape[0]
    flat = lambda t, c: None if t is None else t.reshape(-1, c)  # noqa: E731
    ref = block_reference(flat(x, k), w.to(x.dtype), b, g, h, eps, act, flat(r, n), flat(gy, n), normed)
    hr = 0.0 if x.dtype == torch.float32 else HALF[x.dtype]
    ask = [(kk, t) for kk, t in leaf.items() if t is not None]
    grads = dict(zip([kk for kk, _ in ask], torch.autograd.grad(y, [t for _, t in ask], gy)))
    got = {"y": y.detach(), "gx": grads["x"], "gw": grads["w"], "gb": grads.get("b"), "gg": grads.get("g"), "gh": grads.get("h")}
    for name, t in got.items():
        if t is None or name not in ref:
            continue
        v, c, rd = ref[name]
        close(t.reshape(v.shape), v, v.abs() * HALF[t.dtype] + c * 2.0 ** -24 + rd * hr * 1.01 + 1e-30, f"{what} {name}")
    for kk, t in ask:
        assert grads[kk].shape == t.shape and grads[kk].dtype == t.dtype
    if r is not None:
        assert torch.equal(grads["r"], gy)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("m,k,n,act", [(1, 4, 8, "silu"), (3, 128, 128, "silu"), (64, 33, 17, "elu"), (130, 97, 65, "silu"), (100, 128, 100, "elu"),
                                       (257, 384, 128, "silu"), (1000, 64, 193, "silu"), (2967, 128, 128, "elu"), (300, 200, 256, "silu"),
                                       (129, 96, 257, "silu"), (64, 300, 513, "elu"), (200, 512, 512, "silu"), (33, 1000, 48, "none"),
                                       (40003, 32, 40, "silu")])
def test_linear_blocks(dev, dtype, normed, m, k, n, act):
    gen = torch.Generator(device=dev)
    gen.manual_seed(m + k * 5 + n * 11)
    print(f"{'linear_norm_act' if normed else 'linear_act'} {m} x {k} -> {n} {act} {dtype}", flush=True)
    x = grid_values(gen, (m, k), dev, 1.0).add_(0.25).to(dtype)
    w = (torch.rand(n, k, generator=gen, device=dev) * 2 - 1).div_(math.sqrt(k)).to(dtype)
    b = (torch.rand(n, generator=gen, device=dev) * 2 - 1).to(dtype)
    g = grid_values(gen, (n,), dev, 0.3).add_(1.0).to(dtype)
    h = grid_values(gen, (n,), dev, 0.3).to(dtype)
    r, gy = (grid_values(gen, (m, n), dev, 1.0).to(dtype) for _ in range(2))
    block_check(normed, x, w, b, g, h, 1e-5, act, r, gy, f"{m}x{k}->{n}") if normed else block_check(False, x, w, b, None, None, 0.0, act, r, gy, f"{m}x{k}->{n}")
    if m <= 300:
        block_check(normed, x, w, None, None, None, 1e-3, act, None, gy, f"{m}x{k}->{n} plain")


@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_linear_blocks_strides_and_parameter_types(dev, dtype, normed):
    gen = torch.Generator(device=dev)
    gen.manual_seed(9)
    big = grid_values(gen, (260, 300), dev, 1.0).to(dtype)
    n = 72
    par = [grid_values(gen, s, dev, 0.5) for s in ((n, 100), (n,), (n,), (n,))]
    r, gy = grid_values(gen, (260, n), dev, 1.0).to(dtype), grid_values(gen, (260, n), dev, 1.0).to(dtype)

    def go(x, p, r, gy, what):
        block_check(normed, x, p[0], p[1], p[2] if normed else None, p[3] if normed else None, 1e-5, "silu", r, gy, what)
    same = [t.to(dtype) for t in par]
    for off in (0, 8, 3):
        go(big[:, off:off + 100], same, r, gy, f"slice {off}")
    go(big[::2, :100], same, r[::2], gy[::2], "every second row")
    go(big[:100].t()[:260], same, r, gy, "transposed x") if big[:100].t().shape[0] >= 260 else None
    go(big[:1, :100].expand(50, 100), same, r[:50], gy[:50], "one row expanded")
    go(big[:, :100], [same[0].t().contiguous().t(), *same[1:]], r, gy, "transposed weight")
    go(big[:, :100], [torch.cat((same[0], same[0]), 1)[:, 50:150], *same[1:]], r, gy, "weight slice")
    go(big[:, :100], par, r, gy, "f32 parameters")                                      # (grid values: their 16-bit copies are the same numbers)
    go(big[:240, :100].reshape(2, 3, 40, 100), same, r[:240].reshape(2, 3, 40, n), gy[:240].reshape(2, 3, 40, n), "four dims")
    go(big[0, :100], same, r[0], gy[0], "one row, one dim")


@pytest.mark.parametrize("normed", [False, True])
def test_linear_blocks_rows_do_not_mix(dev, normed):
    """infinities and NaN in one row stay in that row (forward and dX); padding columns of odd widths hold nothing"""
    from pygho_amd import _ops
    gen = torch.Generator(device=dev)
    gen.manual_seed(10)
    for dtype in DTYPES:
        for k, n in ((128, 128), (97, 65), (40, 300)):
            x = torch.randn(150, k, generator=gen, device=dev).to(dtype)
            w, b, g, h = (torch.randn(s, generator=gen, device=dev).to(dtype) for s in ((n, k), (n,), (n,), (n,)))
            gy = torch.randn(150, n, generator=gen, device=dev).to(dtype)
            call = (lambda t: _ops.linear_norm_act(t, w, b, g, h, 1e-5, "silu")) if normed else (lambda t: _ops.linear_act(t, w, b, "silu"))

            def both(t):
                t = t.clone().requires_grad_(True)
                y = call(t)
                return y.detach(), torch.autograd.grad(y, t, gy)[0]
            clean = both(x)
            dirty = x.clone()
            dirty[5, k - 1], dirty[70, 0], dirty[149, k // 2] = float("inf"), float("nan"), float("-inf")
            got = both(dirty)
            keep = torch.ones(150, dtype=torch.bool, device=dev)
            keep[[5, 70, 149]] = False
            for a, c in zip(got, clean):
                assert torch.equal(a[keep], c[keep]) and bool((~torch.isfinite(a[~keep])).any(1).all())


def test_linear_blocks_no_rows(dev):
    from pygho_amd import _ops
    for n in (64, 300):
        x = torch.zeros((0, 40), device=dev, requires_grad=True)
        p = [torch.ones(s, device=dev, requires_grad=True) for s in ((n, 40), (n,), (n,), (n,))]
        for y, ask in ((_ops.linear_act(x, p[0], p[1], "silu"), [x, *p[:2]]), (_ops.linear_norm_act(x, *p, act="silu"), [x, *p])):
            grads = torch.autograd.grad(y, ask, torch.zeros_like(y))
            assert y.shape == (0, n) and all(t.shape == a.shape and not t.any() for t, a in zip(grads, ask))


@pytest.mark.parametrize("normed", [False, True])
def test_linear_blocks_gradients_against_differences(dev, normed):
    """as for layer_norm_act: central differences of the kernel's own f32 forward"""
    from pygho_amd import _ops
    gen = torch.Generator(device=dev)
    gen.manual_seed(11)
    for act in ("none", "silu", "elu"):
        t = [torch.randn(s, generator=gen, device=dev) * sc for s, sc in (((60, 40), 1.0), ((56, 40), 0.2), ((56,), 0.5), ((60, 56), 1.0), ((56,), 1.0),
                                                                         ((56,), 1.0))][:6 if normed else 4]
        gy = torch.randn(60, 56, generator=gen, device=dev)

        def f(a):
            return _ops.linear_norm_act(a[0], a[1], a[2], a[4], a[5], 1e-5, act, residual=a[3]) if normed else _ops.linear_act(a[0], a[1], a[2], act, residual=a[3])
        leaves = [v.clone().requires_grad_(True) for v in t]
        grads = torch.autograd.grad(f(leaves), leaves, gy)
        for i in range(len(t)):
            d = torch.randn(t[i].shape, generator=gen, device=dev)
            v = [float((f([u + s * d if j == i else u for j, u in enumerate(t)]).double() * gy.double()).sum()) for s in (2.0 ** -8, -2.0 ** -8)]
            diff, want = (v[0] - v[1]) / 2.0 ** -7, float((grads[i].double() * d.double()).sum())
            assert abs(diff - want) < 4e-3 * float(grads[i].double().norm() * d.double().norm()) / math.sqrt(d.numel()) + 4e-2, (act, i, diff, want)


@pytest.mark.parametrize("normed", [False, True])
def test_linear_blocks_rows_counted_on_the_device(dev, normed):
    from pygho_amd import _ops
    gen = torch.Generator(device=dev)
    gen.manual_seed(12)
    for dtype in DTYPES:
        for k, n in ((128, 128), (40, 72), (64, 300)):
            w, b, g, h = (torch.randn(s, generator=gen, device=dev).div_(4).to(dtype).requires_grad_(True) for s in ((n, k), (n,), (n,), (n,)))
            for true, cap in ((0, 64), (1, 50), (700, 1000), (1000, 1001), (5000, 40000), (33000, 70000)):
                x, gy = (torch.randn(cap, s, generator=gen, device=dev).to(dtype) for s in (k, n))
                x[true:] = float("nan")
                gy[true:] = float("inf")

                def f(t):
                    return _ops.linear_norm_act(t, w, b, g, h, 1e-5, "silu") if normed else _ops.linear_act(t, w, b, "silu")
                ask = [w, b] + ([g, h] if normed else [])
                xe = x[:true].clone().requires_grad_(True)
                want = torch.autograd.grad(f(xe), [xe, *ask], gy[:true].clone())
                xc = x.requires_grad_(True)
                with _ops.row_families({cap: torch.tensor([true], dtype=torch.int32, device=dev)}):
                    got = torch.autograd.grad(f(xc), [xc, *ask], gy)
                assert torch.equal(got[0][:true], want[0]), (dtype, k, n, true, cap)
                for a, c, name in zip(got[1:], want[1:], "wbgh"):
                    assert torch.equal(a, c), (dtype, k, n, true, cap, name)


def test_linear_blocks_refusals(dev):
    from pygho_amd import _ops
    x, w, b = torch.randn(4, 8, device=dev), torch.randn(5, 8, device=dev), torch.randn(5, device=dev)
    for f in (_ops.linear_act, _ops.linear_norm_act):
        for kw, exc in ((dict(x=x, weight=w, act="tanh"), ValueError), (dict(x=x.double(), weight=w.double()), TypeError),
                        (dict(x=x, weight=w[:, :7]), ValueError), (dict(x=x, weight=w[0]), ValueError), (dict(x=x, weight=w[:0]), ValueError),
                        (dict(x=x, weight=w.half()), TypeError), (dict(x=x.half(), weight=w.bfloat16()), TypeError),
                        (dict(x=x, weight=w, bias=b[:3]), ValueError), (dict(x=x, weight=w, residual=x), ValueError),
                        (dict(x=x, weight=w, residual=torch.zeros(4, 5, device=dev).half()), TypeError), (dict(x=x[:, :0], weight=w[:, :0]), ValueError),
                        (dict(x=x.cpu(), weight=w), RuntimeError), (dict(x=x, weight=w.cpu()), RuntimeError)):
            with pytest.raises(exc):
                f(**kw)
    for kw in (dict(norm_weight=b[:4]), dict(norm_bias=b[:4]), dict(eps=-1.0)):
        with pytest.raises(ValueError):
            _ops.linear_norm_act(x, w, b, **kw)
    x = x.requires_grad_(True)
    g, = torch.autograd.grad(_ops.linear_norm_act(x, w, b, b, b, act="silu").square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), x)
