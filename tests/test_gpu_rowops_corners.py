"""
The row-wise MLP operators (pygho_amd/rowops.py) in their corners: deep activations, 16-bit pre-activations beyond the type's range, infinities in the
last row, rows counted on the device under more than two dims, prediction with parameters that could be trained, modules that the fused MLP has to leave alone.

Tolerances: a result is rounded once (half a step of its type, HALF) after f32 arithmetic; what the f32 part adds is stated at each test.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}      # half of the smallest step of each type
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.device("cuda:0")


def same(got, want, tol, what):
    """|got - want| <= tol, infinities and NaN in the same places"""
    got = got.double()
    ok = ((got - want).abs() <= tol) | (got == want) | (torch.isnan(got) & torch.isnan(want))
    if not bool(ok.all()):
        i = int((~ok).flatten().nonzero()[0])
        raise AssertionError(f"{what}: {int((~ok).sum())} of {ok.numel()} off, first at {i}: got {got.flatten()[i].item()!r}, want {want.flatten()[i].item()!r}")


# ---- the slope of elu far below zero ------------------------------------------------------------------------------------------------
# exp(u) in f32 for u exact: the rounding of u log2(e) moves the exponential by |u| 2^-24 relative, exp2 / expf and the product by 2^-22 at most;
# the sums are of terms of one sign, at most 400 of them in any order: (|u| + 4 + 400) 2^-24 covers all of it
DEEP = 512 * 2.0 ** -24


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [16, 64, 100, 128, 256, 300, 512])
def test_elu_slope_far_below_zero_linear(dev, dtype, n):
    """W = identity: z is x and gx the gradient of z itself.  expm1(z) + 1 would be 0 below -17 and 1e-3 off at -12"""
    from pygho_amd import _ops
    m = 90
    x = -8.0 - 0.25 * (torch.arange(m * n, device=dev) % 89).reshape(m, n)                        # -8 .. -30, exact in every type
    x, w, b = x.to(dtype), torch.eye(n, device=dev, dtype=dtype), torch.zeros(n, device=dev)
    gy = (1.0 + (torch.arange(m * n, device=dev) % 4).reshape(m, n)).to(dtype)
    t = [x.requires_grad_(True), w.requires_grad_(True), b.requires_grad_(True)]
    gx, gw, gb = torch.autograd.grad(_ops.linear_act(*t, act="elu"), t, gy)
    dz = gy.double() * torch.exp(x.detach().double())
    same(gx, dz, dz * (2 * HALF[dtype] + DEEP) + 2 * TINY[dtype], f"gx {n}")                         # (16-bit: dz is rounded, then the result)
    same(gb, dz.sum(0), dz.sum(0) * (HALF[torch.float32] + DEEP), f"gb {n}")
    want, size = dz.t() @ x.detach().double(), dz.t() @ x.detach().double().abs()
    same(gw, want, size * (2 * HALF[dtype] + DEEP) + m * 40 * TINY[dtype], f"gw {n}")                # dz of f16 may be subnormal: m rows of |x| <= 30


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("c", [16, 100, 128, 257, 1000, 2056])
def test_elu_slope_far_below_zero_norm(dev, dtype, c):
    """a norm whose weight is zero hands its bias to the activation: gbias = sum gy exp(bias)"""
    from pygho_amd import _ops
    m = 90
    h = (-8.0 - 0.25 * (torch.arange(c, device=dev) % 89)).requires_grad_(True)
    g = torch.zeros(c, device=dev, requires_grad=True)
    x = torch.randn(m, c, generator=torch.Generator(device=dev).manual_seed(c), device=dev).to(dtype)
    gy = (1.0 + (torch.arange(m * c, device=dev) % 4).reshape(m, c)).to(dtype)
    want = (gy.double() * torch.exp(h.detach().double())).sum(0)
    gh, = torch.autograd.grad(_ops.layer_norm_act(x, g, h, act="elu"), h, gy)
    same(gh, want, want * (HALF[torch.float32] + DEEP), f"layer_norm_act {c}")
    w = torch.randn(c, 32, generator=torch.Generator(device=dev).manual_seed(c), device=dev).to(dtype)
    gh, = torch.autograd.grad(_ops.linear_norm_act(x[:, :16].repeat(1, 2), w, None, g, h, act="elu"), h, gy)
    same(gh, want, want * (HALF[torch.float32] + DEEP), f"linear_norm_act {c}")


# ---- a pre-activation that is kept in 16 bits ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("act", ["silu", "elu", "relu"])
@pytest.mark.parametrize("k,n", [(128, 128), (256, 256), (300, 300), (512, 512)])
def test_f16_pre_activations_beyond_the_type(dev, k, n, act):
    """|z| of 2 or 4 times f16's largest value: the slope is 0 or 1, in the forms that keep z as in those that form it again; dz is gy or 0 and every
    sum below exact.  An infinity that the input holds stays one"""
    from pygho_amd import _ops
    m = 40
    sign = torch.where(torch.arange(n, device=dev) % 2 == 0, 1.0, -1.0)
    x = torch.full((m, k), 1024.0, device=dev, dtype=torch.float16)
    w = (sign[:, None] * (1.0 if k <= 256 else 0.5)).expand(n, k).contiguous().half()
    gy = (torch.arange(m * n, device=dev) % 3 - 1).reshape(m, n).half()
    x.requires_grad_(True), w.requires_grad_(True)
    y = _ops.linear_act(x, w, None, act)
    gx, gw = torch.autograd.grad(y, (x, w), gy)
    z = x.detach().double() @ w.detach().double().t()
    assert float(z.abs().min()) > 65504 * 1.9
    dz = gy.double() * (z > 0)
    low = {"silu": 0.0, "elu": -1.0, "relu": 0.0}[act]
    assert torch.equal(y.detach(), torch.where(z > 0, z, torch.full_like(z, low)).half())
    assert torch.equal(gx, (dz @ w.detach().double()).half())
    assert torch.equal(gw, (dz.t() @ x.detach().double()).half())
    if act == "silu":
        bad = x.detach().clone()
        bad[3, 5] = float("inf")
        bad.requires_grad_(True)
        gx, = torch.autograd.grad(_ops.linear_act(bad, w.detach(), None, act), bad, torch.ones_like(gy))
        assert bool(torch.isnan(gx[3]).all()) and bool(torch.isfinite(gx[:3]).all()) and bool(torch.isfinite(gx[4:]).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["silu", "elu"])
@pytest.mark.parametrize("m,k,n", [(1, 244, 344), (1, 512, 512), (2, 300, 300), (1, 256, 256), (1, 128, 128), (3, 600, 100), (1, 40, 700)])
def test_the_slope_is_that_of_the_unrounded_pre_activation(dev, m, k, n, act, dtype):
    """few rows, so that no average hides it: gx and gw within one rounding of dz and one of the result (the bounds of `block_reference`), in the forms
    that keep z as in those that form it again.  A z rounded to bf16 moves silu's slope by up to 2^-8"""
    from test_gpu_rowops import block_check, grid_values
    gen = torch.Generator(device=dev).manual_seed(m + k + n)
    x = grid_values(gen, (m, k), dev, 1.0).add_(0.25).to(dtype)
    w = (torch.rand(n, k, generator=gen, device=dev) * 2 - 1).div_(k ** 0.5).to(dtype)
    gy = grid_values(gen, (m, n), dev, 1.0).to(dtype)
    block_check(False, x, w, None, None, None, 0.0, act, None, gy, f"{m} x {k} -> {n}")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_a_caller_of_the_c_entry_may_keep_z_in_the_rows_type(dev, dtype):
    """both storages of z through the C entry, with a z beyond f16: values and slopes of an exact product"""
    from pygho_amd import _ops
    from pygho_amd._native import DTYPE_CODE, check, lib, ptr, stream_ptr
    m, k, n, code, silu = 40, 512, 512, DTYPE_CODE[dtype], _ops.ROW_ACT_CODE["silu"]
    sign = torch.where(torch.arange(n, device=dev) % 2 == 0, 1.0, -1.0)
    x, w = torch.full((m, k), 1024.0, device=dev, dtype=dtype), (0.5 * sign[:, None]).expand(n, k).contiguous().to(dtype)
    gy = (torch.arange(m * n, device=dev) % 3 - 1).reshape(m, n).to(dtype)
    want = ((gy.double() * (sign > 0)) @ w.double()).to(dtype)
    assert int(lib().pygho_linear_act_keeps(k, n, 0, silu, code)) == 1
    nbytes = int(lib().pygho_linear_act_bwd_workspace(m, k, n, 0, silu, code))
    for flag, zt in ((0, dtype), (0x100, torch.float32)):
        y, gx, ws = torch.empty_like(gy), torch.empty_like(x), torch.empty(nbytes, dtype=torch.uint8, device=dev)
        z = torch.full((m + 1, n), 7.0, dtype=zt, device=dev)
        check(lib().pygho_linear_act(ptr(y), ptr(z), ptr(x), k, ptr(w), k, None, 0, 0, None, None, 0, 0.0, None, 0, m, k, n, silu | flag, code, stream_ptr(dev)),
              "linear_act")
        full = 1024.0 * 0.5 * k * sign
        if zt == torch.float16:
            full = full.clamp(-65504.0, 65504.0)
        assert torch.equal(z[:m].double(), full.double().expand(m, n)) and bool((z[m] == 7.0).all())
        check(lib().pygho_linear_act_bwd(ptr(gx), None, 0, None, 0, None, 0, None, 0, ptr(z), ptr(x), k, ptr(w), k, None, 0, 0, None, None, 0, 0.0, ptr(gy), n, m,
                                         None, k, n, silu | flag, code, ptr(ws), nbytes, stream_ptr(dev)), "linear_act_bwd")
        assert torch.equal(gx, want), (flag, zt)


# ---- infinities in the last row ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k,n", [(128, 128), (64, 64), (96, 112), (100, 36), (384, 128), (256, 256), (512, 512)])
@pytest.mark.parametrize("m", [1, 17, 333, 2000])
def test_an_infinity_in_the_last_row_counts_once(dev, dtype, m, k, n):
    """the weight's gradient is infinite where that row's dz is not zero, NaN where it is (0 * inf), and finite in the other columns -- whatever a
    launch does with the lanes behind the last row.  Small integers: everything finite is exact"""
    from pygho_amd import _ops
    gen = torch.Generator(device=dev).manual_seed(m + k + n)
    x = torch.randint(-2, 3, (m, k), generator=gen, device=dev).to(dtype)
    w = (torch.randint(0, 2, (n, k), generator=gen, device=dev) * 2 - 1).to(dtype)              # no zeros: z of that row is +-inf, never NaN
    gy = torch.randint(1, 3, (m, n), generator=gen, device=dev).to(dtype)
    x[m - 1, 7] = float("inf")
    z = x.double() @ w.double().t()
    dz = gy.double() * (z > 0)
    t = [x.requires_grad_(True), w.requires_grad_(True)]
    gw, = torch.autograd.grad(_ops.linear_act(*t, act="relu"), t[1:], gy)
    want = dz.t() @ x.detach().double()
    assert bool(torch.isinf(want[:, 7]).any()) and bool(torch.isnan(want[:, 7]).any()) and bool(torch.isfinite(want[:, :7]).all())
    same(gw, want.to(dtype).double(), torch.zeros_like(want), f"{m} x {k} -> {n}")


# ---- rows counted on the device: the family is named by the extent of dim 0 ------------------------------------------------------------
def calls(_ops, k, n, gen, dev, dtype):
    p = [torch.randn(s, generator=gen, device=dev).div_(4).to(dtype).requires_grad_(True) for s in ((n, k), (n,), (n,), (n,), (k,), (k,))]
    return [(lambda t: _ops.layer_norm_act(t, p[4], p[5], act="silu"), k, p[4:]), (lambda t: _ops.linear_act(t, p[0], p[1], "silu"), n, p[:2]),
            (lambda t: _ops.linear_norm_act(t, p[0], p[1], p[2], p[3], act="silu"), n, p[:4])]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("inner", [(3,), (2, 5), (1,)])
def test_device_row_counts_under_more_dims(dev, dtype, inner):
    """x (capacity, j, .., C) with `true` of its first extent in use: the bits of the exactly sized call, whatever the rest holds"""
    from pygho_amd import _ops
    gen = torch.Generator(device=dev).manual_seed(len(inner))
    for k, n in ((128, 128), (40, 72), (64, 300)):
        for true, cap in ((0, 64), (1, 50), (700, 1001), (1001, 1001)):
            for f, width, par in calls(_ops, k, n, gen, dev, dtype):
                x = torch.randn((cap, *inner, k), generator=gen, device=dev).to(dtype)
                gy = torch.randn((cap, *inner, width), generator=gen, device=dev).to(dtype)
                x[true:], gy[true:] = float("nan"), float("inf")
                xe = x[:true].clone().requires_grad_(True)
                want = torch.autograd.grad(f(xe), [xe, *par], gy[:true].clone())
                x.requires_grad_(True)
                with _ops.row_families({cap: torch.tensor([true], dtype=torch.int32, device=dev)}):
                    got = torch.autograd.grad(f(x), [x, *par], gy)
                assert torch.equal(got[0][:true], want[0]), (k, n, true, cap)
                assert all(torch.equal(a, b) for a, b in zip(got[1:], want[1:])), (k, n, true, cap)


@pytest.mark.parametrize("dtype", DTYPES)
def test_tensors_whose_other_extents_meet_a_capacity(dev, dtype):
    """rows of (a, b, C) with a b = a capacity, or a single row of that many channels, belong to no family: nothing is cut off"""
    from pygho_amd import _ops
    gen = torch.Generator(device=dev).manual_seed(1)
    for shape, cap in (((20, 50, 64), 1000), ((5, 50, 64), 50), ((64,), 64), ((7, 64), 64)):
        for f, width, par in calls(_ops, 64, 72, gen, dev, dtype):
            x = torch.randn(shape, generator=gen, device=dev).to(dtype).requires_grad_(True)
            gy = torch.randn(shape[:-1] + (width,), generator=gen, device=dev).to(dtype)
            want = torch.autograd.grad(f(x), [x, *par], gy)
            with _ops.row_families({cap: torch.tensor([3], dtype=torch.int32, device=dev)}):
                got = torch.autograd.grad(f(x), [x, *par], gy)
            assert all(torch.equal(a, b) for a, b in zip(got, want)), (shape, cap)


def test_device_row_counts_under_more_dims_captured(dev):
    """the scaled count is read at every replay"""
    from pygho_amd import _ops
    gen = torch.Generator(device=dev).manual_seed(2)
    cap, count = 600, torch.tensor([600], dtype=torch.int32, device=dev)
    x = torch.randn(cap, 3, 64, generator=gen, device=dev).bfloat16().requires_grad_(True)
    w = torch.randn(72, 64, generator=gen, device=dev).bfloat16().requires_grad_(True)
    gy = torch.randn(cap, 3, 72, generator=gen, device=dev).bfloat16()

    def step(xx, gg):
        return torch.autograd.grad(_ops.linear_act(xx, w, None, "silu"), (xx, w), gg)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), _ops.row_families({cap: count}):
        step(x, gy)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with _ops.row_families({cap: count}), torch.cuda.graph(g):
        out = step(x, gy)
    for true in (600, 17, 1, 0, 333):
        count.fill_(true)
        g.replay()
        torch.cuda.synchronize()
        xe = x.detach()[:true].clone().requires_grad_(True)
        want = step(xe, gy[:true].clone())
        assert torch.equal(out[0][:true], want[0]) and torch.equal(out[1], want[1]), true


# ---- prediction with parameters that could be trained --------------------------------------------------------------------------------
def peak(f):
    f()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    base = torch.cuda.memory_allocated()
    out = f()
    torch.cuda.synchronize()
    return torch.cuda.max_memory_allocated() - base, out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_prediction_keeps_no_pre_activation(dev, dtype):
    """512 -> 512 with an activation is the form that keeps z for a gradient: without one only the output is allocated"""
    from pygho_amd import _ops
    x = torch.randn(20000, 512, device=dev).to(dtype)
    w, b = torch.nn.Parameter(torch.randn(512, 512, device=dev).to(dtype)), torch.nn.Parameter(torch.randn(512, device=dev).to(dtype))
    size = x.numel() * x.element_size()

    def call():
        return _ops.linear_act(x, w, b, "silu")
    trained, y = peak(call)
    assert trained >= 2 * size and y.requires_grad
    with torch.no_grad():
        spent, p = peak(call)
    assert torch.equal(p, y.detach()) and not p.requires_grad and size <= spent < 1.1 * size
    with torch.inference_mode():
        spent, p = peak(call)
    assert torch.equal(p, y.detach()) and size <= spent < 1.1 * size
    # the residual alone needs a gradient: gy is all of it
    spent, p = peak(lambda: _ops.linear_act(x, w.detach(), b.detach(), "silu", residual=x.detach().requires_grad_(True)))
    assert p.requires_grad and spent < 1.1 * size


# ---- what the fused MLP leaves to the stock modules ------------------------------------------------------------------------------------
@pytest.mark.parametrize("norm", ["ln", "none"])
def test_fused_mlp_leaves_other_types_to_the_stock_modules(dev, norm):
    from pygho_amd.honn.utils import MLP
    torch.manual_seed(0)
    stock, fused = (MLP(40, 24, 2, True, norm=norm, act="silu", fused=f).to(dev).double() for f in (False, True))
    fused.load_state_dict(stock.state_dict())
    x, r = torch.randn(33, 40, device=dev, dtype=torch.float64), torch.randn(33, 24, device=dev, dtype=torch.float64)
    out = []
    for m in (stock, fused):
        xx = x.clone().requires_grad_(True)
        y = m(xx, residual=r)
        out.append((y.detach(), *torch.autograd.grad(y.sum(), [xx, *m.parameters()])))
    assert out[1][0].dtype == torch.float64 and all(torch.equal(a, b) for a, b in zip(*out))


def test_fused_mlp_runs_hooks_and_modules_of_the_users_own(dev):
    """a hook on an inner module, a Linear whose forward is another, a weight under a parametrization: their code runs"""
    from pygho_amd.honn.utils import MLP
    torch.manual_seed(0)
    x = torch.randn(33, 40, device=dev)

    def model():
        torch.manual_seed(1)
        return MLP(40, 40, 2, True, norm="ln", act="silu", fused=True).to(dev)
    plain, seen = model()(x), []
    for i in range(6):
        m = model()
        seen.clear()
        handle = m.lins[i].register_forward_hook(lambda mod, args, out: seen.append(type(mod).__name__))
        try:
            assert float((m(x) - plain).abs().max()) < 1e-5 and seen       # (activations are shared between the blocks: once or twice)
        finally:
            handle.remove()
        assert torch.equal(m(x), plain)
    m = model()
    m.lins[1].norm.register_forward_pre_hook(lambda mod, args: seen.append("norm"))
    m(x)
    assert seen[-1] == "norm"

    class Doubled(torch.nn.Linear):
        def forward(self, t):
            return 2.0 * super().forward(t)
    m = model()
    own = Doubled(40, 40).to(dev)
    own.load_state_dict(m.lins[0].state_dict())
    m.lins[0] = own
    want = m.lins[5](m.lins[4](m.lins[3](m.lins[2](m.lins[1](own(x))))))
    assert float((m(x) - want).abs().max()) < 1e-5
    m = model()
    torch.nn.utils.parametrizations.weight_norm(m.lins[3])
    assert float((m(x) - plain).abs().max()) < 1e-5


def test_fused_mlp_on_rows_far_apart(dev):
    """rows 2^27 bytes apart, which the operators refuse: the MLP takes a copy.  A gradient that arrives that way as well"""
    from pygho_amd import _ops
    from pygho_amd.honn.utils import MLP
    torch.manual_seed(0)
    m = MLP(128, 128, 1, True, norm="ln", act="silu", fused=True).to(dev)
    x, gy = torch.randn(2, 128, device=dev), torch.randn(2, 128, device=dev)
    room = torch.empty((1 << 25) + 1024, device=dev)
    far, gfar = room.as_strided((2, 128), (1 << 25, 1)), room.as_strided((2, 128), (1 << 25, 1), 512)
    far.copy_(x)
    gfar.copy_(gy)
    with pytest.raises(RuntimeError, match="strides"):
        _ops.linear_act(far, m.lins[0].weight)
    assert torch.equal(m(far, residual=far), m(x, residual=x))
    t = x.clone().requires_grad_(True)
    got, want = (torch.autograd.grad(m(t), [t, *m.parameters()], g) for g in (gfar, gy))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---- only what is asked for ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("norm", [0, 1])
@pytest.mark.parametrize("k,n", [(128, 128), (96, 112), (384, 128), (100, 36), (256, 256), (40, 300), (512, 512)])
def test_the_workspace_of_a_call_holds_it(dev, dtype, norm, k, n):
    """the C entry with just the bytes that the query for this call names, for every subset of gradients and both activations' plans: nothing is
    written behind them, and the values are those of the call with every gradient in the largest workspace"""
    import itertools
    from pygho_amd import _ops
    from pygho_amd._native import DTYPE_CODE, check, lib, ptr, stream_ptr
    gen = torch.Generator(device=dev).manual_seed(k + n)
    m, code, guard = 777, DTYPE_CODE[dtype], 1 << 14
    x, w, b, g, h, gy = (torch.randn(s, generator=gen, device=dev).div_(4).to(dtype) for s in ((m, k), (n, k), (n,), (n,), (n,), (m, n)))
    names = ("gx", "gw", "gb") + (("gg", "gh") if norm else ())
    for act in (_ops.ROW_ACT_CODE["none"], _ops.ROW_ACT_CODE["silu"]):
        keeps = int(lib().pygho_linear_act_keeps(k, n, norm, act, code))
        y, z = torch.empty_like(gy), torch.empty((m, n), dtype=torch.float32 if keeps == 2 else dtype, device=dev)
        check(lib().pygho_linear_act(ptr(y), ptr(z), ptr(x), k, ptr(w), k, ptr(b), code, norm, ptr(g), ptr(h), code, 1e-5, None, 0, m, k, n, act, code,
                                     stream_ptr(dev)), "linear_act")

        def backward(ask, nbytes):
            out = {name: torch.full(s, 7.0, dtype=dtype, device=dev) for name, s in (("gx", (m, k)), ("gw", (n, k)), ("gb", (n,)), ("gg", (n,)), ("gh", (n,)))
                   if name in ask}
            if nbytes is None:
                nbytes = int(lib().pygho_linear_act_bwd_workspace_for(ptr(out.get("gx")), "gw" in ask, "gb" in ask, ptr(x), k, ptr(gy), n, m, k, n, norm,
                                                                      act, code))
                assert nbytes <= int(lib().pygho_linear_act_bwd_workspace(m, k, n, norm, act, code))
            ws = torch.full((nbytes + guard,), 0xA5, dtype=torch.uint8, device=dev)
            p = {name: ptr(out.get(name)) for name in ("gx", "gw", "gb", "gg", "gh")}
            check(lib().pygho_linear_act_bwd(p["gx"], p["gw"], code, p["gb"], code, p["gg"], code, p["gh"], code, ptr(z) if keeps else None, ptr(x), k, ptr(w), k,
                                             ptr(b), code, norm, ptr(g), ptr(h), code, 1e-5, ptr(gy), n, m, None, k, n, act, code, ptr(ws), nbytes,
                                             stream_ptr(dev)), "linear_act_bwd")
            assert bool((ws[nbytes:] == 0xA5).all()), (act, ask)
            return out
        want = backward(names, int(lib().pygho_linear_act_bwd_workspace(m, k, n, norm, act, code)))
        for pick in itertools.product((False, True), repeat=len(names)):
            ask = [name for name, f in zip(names, pick) if f]
            got = backward(ask, None)
            for name in ask:
                # dX without an activation or a norm is gy . W in either of two launches: the same n products in another order, each off by at most
                # n 2^-24 of their absolute sum and rounded once (two of 128 x 128 bf16 values differ in the last bit).  With one: the same order
                if name == "gx" and not norm and act == _ops.ROW_ACT_CODE["none"]:
                    v = want[name].double()
                    same(got[name], v, v.abs() * 2 * HALF[dtype] + 2 * n * 2.0 ** -24 * (gy.double().abs() @ w.double().abs()) + TINY[dtype], f"{ask} gx")
                elif name == "gx":
                    assert torch.equal(got[name], want[name]), (act, ask)
                else:                                           # other slabs: the rows in another order, chains of at most 256 sums of m terms below 1 on average
                    v = want[name].double()
                    same(got[name], v, v.abs() * 2 * HALF[dtype] + 256 * 2.0 ** -24 * m, f"{act} {ask} {name}")
