"""
The row-wise linear operators where one launch form ends and the next begins: every subset of gradients, ragged edges of the largest tiles,
the longest row strides, 16-bit rows at odd addresses.  Small integers throughout: every partial sum in f32 is exact in any order, so that the
only rounding is the last one and results are compared bit for bit.
"""
import itertools

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.device("cuda:0")


def integers(gen, shape, dev, most, dtype):
    return torch.randint(-most, most + 1, shape, generator=gen, device=dev).to(dtype)


def exact(x, w, b, gy):
    """relu(x W^T + b): output and gradients in 64 bits"""
    z = x.double() @ w.double().t() + b.double()
    dz = gy.double() * (z > 0)
    return torch.relu(z), dz @ w.double(), dz.t() @ x.double(), dz.sum(0)


# (m, k, n): the fused gradient, streams with dX in the same launch and without it, x in registers, tiles
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,n", [(333, 128, 128), (333, 64, 64), (333, 96, 112), (333, 384, 128), (333, 100, 36), (333, 256, 256), (200, 512, 512)])
def test_every_subset_of_gradients(dev, dtype, m, k, n):
    from pygho_amd import _ops
    gen = torch.Generator(device=dev)
    gen.manual_seed(m + k + n)
    x, w, b, gy = (integers(gen, s, dev, most, dtype) for s, most in (((m, k), 2), ((n, k), 2), ((n,), 9), ((m, n), 2)))
    y, *want = exact(x, w, b, gy)
    for need in itertools.product((False, True), repeat=3):
        if not any(need):
            continue
        leaves = [t.clone().requires_grad_(f) for t, f in zip((x, w, b), need)]
        out = _ops.linear_act(*leaves, act="relu")
        assert torch.equal(out.detach(), y.to(dtype))
        got = torch.autograd.grad(out, [t for t in leaves if t.requires_grad], gy)
        for g, v in zip(got, [v for v, f in zip(want, need) if f]):
            assert torch.equal(g, v.to(dtype)), (need, g.shape)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,k,n", [(333, 128, 128), (333, 96, 112), (200, 512, 512), (100, 40, 24)])
def test_every_subset_of_gradients_with_a_norm(dev, dtype, m, k, n):
    from pygho_amd import _ops
    from test_gpu_rowops import HALF, block_reference, close      # (the bounds are derived there)
    gen = torch.Generator(device=dev)
    gen.manual_seed(m + k + n)
    x, w, b, g, h = t = [v.to(dtype) for v in (
        torch.randn(m, k, generator=gen, device=dev), torch.randn(n, k, generator=gen, device=dev) / k ** 0.5, torch.randn(n, generator=gen, device=dev),
        torch.rand(n, generator=gen, device=dev) + 0.5, torch.randn(n, generator=gen, device=dev))]
    gy = torch.randn(m, n, generator=gen, device=dev).to(dtype)
    ref = block_reference(x, w, b, g, h, 1e-5, "silu", None, gy, True)
    hr = 0.0 if dtype == torch.float32 else HALF[dtype]
    names = ("gx", "gw", "gb", "gg", "gh")
    for need in itertools.product((False, True), repeat=5):
        if not any(need):
            continue
        leaves = [v.clone().requires_grad_(f) for v, f in zip(t, need)]
        got = torch.autograd.grad(_ops.linear_norm_act(*leaves, act="silu"), [v for v in leaves if v.requires_grad], gy)
        for name, grad in zip([v for v, f in zip(names, need) if f], got):
            v, c, rd = ref[name]
            close(grad, v, v.abs() * HALF[dtype] + c * 2.0 ** -24 + rd * hr * 1.01 + 1e-30, f"{need} {name}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,n", [(66001, 512, 320), (66001, 320, 500), (70001, 300, 300), (33000, 512, 512)])
def test_large_tiles_with_ragged_edges(dev, dtype, m, k, n):
    from pygho_amd import _ops
    gen = torch.Generator(device=dev)
    gen.manual_seed(m + k + n)
    x, w, b, gy = (integers(gen, s, dev, most, dtype) for s, most in (((m, k), 1), ((n, k), 1), ((n,), 9), ((m, n), 1)))
    y, gx, gw, gb = exact(x, w, b, gy)
    assert float(gw.abs().max()) < 2 ** 24 and float(gb.abs().max()) < 2 ** 24
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    out = _ops.linear_act(*leaves, act="relu")
    assert torch.equal(out.detach(), y.to(dtype))
    for g, v in zip(torch.autograd.grad(out, leaves, gy), (gx, gw, gb)):
        assert torch.equal(g, v.to(dtype)), g.shape


def test_long_row_strides(dev):
    """rows just below 2^27 bytes apart: 40 of them reach past every 32-bit offset; 2^27 bytes are refused"""
    from pygho_amd import _ops
    gen = torch.Generator(device=dev)
    gen.manual_seed(1)
    stride = (1 << 26) - 8
    for k, n in ((128, 128), (256, 256), (64, 20), (512, 512)):
        x, w, b, gy = (integers(gen, s, dev, 2, torch.bfloat16) for s in ((40, k), (n, k), (n,), (40, n)))
        y, gx, gw, gb = exact(x, w, b, gy)
        far = torch.empty(39 * stride + 1024, dtype=torch.bfloat16, device=dev)
        fx, fr = far.as_strided((40, k), (stride, 1)), far.as_strided((40, n), (stride, 1), 512)
        fx.copy_(x)
        fr.copy_(gy)
        leaves = [fx.detach().requires_grad_(True), w.clone().requires_grad_(True), b.clone().requires_grad_(True)]
        out = _ops.linear_act(*leaves, act="relu", residual=fr)
        assert torch.equal(out.detach(), (y + gy.double()).to(torch.bfloat16))
        for g, v in zip(torch.autograd.grad(out, leaves, fr), (gx, gw, gb)):
            assert torch.equal(g, v.to(torch.bfloat16)), g.shape
        assert torch.equal(_ops.layer_norm_act(fx, act="silu"), _ops.layer_norm_act(x, act="silu"))
        del far, fx, fr, leaves, out
    x = torch.empty(2 * (1 << 26), dtype=torch.bfloat16, device=dev).as_strided((2, 128), (1 << 26, 1))
    with pytest.raises(RuntimeError, match="strides"):
        _ops.linear_act(x, torch.empty(128, 128, dtype=torch.bfloat16, device=dev))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("k,n", [(128, 128), (129, 127), (256, 256), (512, 320), (64, 20), (7, 3)])
def test_rows_at_odd_addresses(dev, dtype, k, n):
    """x, W, bias, residual and output gradient each start one element past a vector's boundary and have rows of an odd stride"""
    from pygho_amd import _ops
    gen = torch.Generator(device=dev)
    gen.manual_seed(k + n)

    def odd(rows, c):
        v = torch.full((rows * (c + 4 + c % 2 + 1) + 8,), 7.0, dtype=dtype, device=dev)[1:].as_strided((rows, c), (c + 4 + c % 2 + 1, 1))
        v.copy_(integers(gen, (rows, c), dev, 2, dtype))
        return v
    x, w, r, gy = odd(500, k), odd(n, k), odd(500, n), odd(500, n)
    b = odd(1, n)[0]
    y, gx, gw, gb = exact(x, w, b, gy)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    out = _ops.linear_act(*leaves, act="relu", residual=r)
    assert torch.equal(out.detach(), (y + r.double()).to(dtype))
    for g, v in zip(torch.autograd.grad(out, leaves, gy), (gx, gw, gb)):
        assert torch.equal(g, v.to(dtype)), g.shape


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("k,n", [(128, 128), (384, 128), (100, 36), (256, 256), (100, 513), (512, 512), (300, 20)])
@pytest.mark.parametrize("true", [0, 1, 300])
def test_rows_behind_the_device_count_stay_as_they_were(dev, dtype, k, n, true):
    """the C entry with a capacity of 500 rows and the true count on the device: gx behind the count keeps its bytes, what x, gy and z hold
    there (NaN) reaches nothing"""
    from pygho_amd import _ops
    from pygho_amd._native import DTYPE_CODE, check, lib, ptr, stream_ptr
    gen = torch.Generator(device=dev)
    gen.manual_seed(k + n + true)
    cap, code, act = 500, DTYPE_CODE[dtype], _ops.ROW_ACT_CODE["relu"]
    x, w, b, gy = (integers(gen, s, dev, most, dtype) for s, most in (((cap, k), 2), ((n, k), 2), ((n,), 9), ((cap, n), 2)))
    _, gx, gw, gb = exact(x[:true], w, b, gy[:true])
    keeps = int(lib().pygho_linear_act_keeps(k, n, 0, act, code))
    z = (x.double() @ w.double().t() + b.double()).to(dtype) if keeps else None
    for t in (x, gy) + ((z,) if keeps else ()):
        t[true:] = float("nan")
    out, gw2, gb2 = torch.full((cap, k), 77.0, dtype=dtype, device=dev), torch.empty_like(w), torch.empty_like(b)
    count = torch.tensor([true], dtype=torch.int32, device=dev)
    nbytes = int(lib().pygho_linear_act_bwd_workspace(cap, k, n, 0, act, code))
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    check(lib().pygho_linear_act_bwd(ptr(out), ptr(gw2), code, ptr(gb2), code, None, 0, None, 0, ptr(z), ptr(x), k, ptr(w), k, ptr(b), code, 0, None, None,
                                     0, 0.0, ptr(gy), n, cap, ptr(count), k, n, act, code, ptr(ws), nbytes, stream_ptr(dev)), "linear_act_bwd")
    assert bool((out[true:] == 77.0).all())
    assert torch.equal(out[:true], gx.to(dtype)) and torch.equal(gw2, gw.to(dtype)) and torch.equal(gb2, gb.to(dtype))


@pytest.mark.parametrize("k,n", [(128, 128), (256, 130), (520, 130)])
def test_more_elements_than_32_bits_count(dev, k, n):
    """the last rows of 2^31 elements and 2^32 bytes give the bits that they give alone; parameters' gradients of gy that is zero elsewhere too"""
    from pygho_amd import _ops
    gen = torch.Generator(device=dev)
    gen.manual_seed(k)
    m, tail = (1 << 31) // min(k, n) + 100001, 777
    w, b, xt, gt = (integers(gen, s, dev, 2, torch.bfloat16) for s in ((n, k), (n,), (tail, k), (tail, n)))
    x = torch.ones(m, k, dtype=torch.bfloat16, device=dev)
    gy = torch.zeros(m, n, dtype=torch.bfloat16, device=dev)
    x[m - tail:], gy[m - tail:] = xt, gt
    y, gx, gw, gb = exact(xt, w, b, gt)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    out = _ops.linear_act(*leaves, act="relu")
    assert torch.equal(out.detach()[m - tail:], y.to(torch.bfloat16))
    grads = torch.autograd.grad(out, leaves, gy)
    assert torch.equal(grads[0][m - tail:], gx.to(torch.bfloat16)) and not grads[0][: m - tail].any()
    assert torch.equal(grads[1], gw.to(torch.bfloat16)) and torch.equal(grads[2], gb.to(torch.bfloat16))
    del out, grads
    if k == 128:
        ln = _ops.layer_norm_act(x.detach(), act="silu")
        assert torch.equal(ln[m - tail:], _ops.layer_norm_act(xt, act="silu"))
        del ln
        a, = torch.autograd.grad(_ops.layer_norm_act(x, act="elu"), x, gy)
        c, = torch.autograd.grad(_ops.layer_norm_act(xt.requires_grad_(True), act="elu"), xt, gt)
        assert torch.equal(a[m - tail:], c)


def test_small_calls_take_small_workspaces(dev):
    from pygho_amd._native import DTYPE_CODE, lib
    at = [int(lib().pygho_linear_act_bwd_workspace(m, 128, 128, 1, 2, DTYPE_CODE[torch.bfloat16])) for m in (1, 16, 100, 10 ** 5, 10 ** 7)]
    assert at == sorted(at) and at[0] < (1 << 20)
