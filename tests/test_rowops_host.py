"""CPU checks of the row-wise MLP operators: the C entry points refuse bad arguments before any launch, the Python ones refuse CPU tensors."""
import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from pygho_amd import build
    build.build(force=False, verbose=False)
    from pygho_amd import _native
    return _native.lib()


ONE = ctypes.c_void_p(16)       # never dereferenced: the checks fail first
F32, BF16, F16, F64 = 0, 1, 2, 3


def test_layer_norm_refusals(lib):
    def fwd(y=ONE, x=ONE, pdt=BF16, m=5, c=128, eps=1e-5, act=2, dt=BF16):
        return lib.pygho_layer_norm_act(y, x, 128, None, None, pdt, None, 0, m, c, eps, act, dt, None)
    assert fwd(m=0) == 0
    assert fwd(m=-1) == 1 and fwd(c=0) == 1 and fwd(act=4) == 1 and fwd(act=-1) == 1 and fwd(eps=-1.0) == 1 and fwd(eps=float("nan")) == 1
    assert fwd(y=None) == 1 and fwd(x=None) == 1 and b"null" in lib.pygho_last_error()
    assert fwd(dt=F64) == 2 and fwd(pdt=F16) == 2

    def bwd(gx=ONE, gy=ONE, ws=ONE, nbytes=1 << 30, m=5, gdt=BF16, c=128):
        return lib.pygho_layer_norm_act_bwd(gx, ONE, gdt, None, 0, ONE, 128, gy, 128, None, None, BF16, m, None, c, 1e-5, 2, BF16, ws, nbytes, None)
    assert bwd(gy=None) == 1 and bwd(ws=None) == 1 and bwd(gx=None) == 1 and bwd(gdt=F64) == 2 and bwd(m=-1) == 1
    assert bwd(nbytes=16) == 1 and b"workspace" in lib.pygho_last_error()
    assert bwd(ws=ctypes.c_void_p(24)) == 1 and b"workspace" in lib.pygho_last_error()
    assert lib.pygho_layer_norm_act_bwd_workspace(0, 128) == 0
    assert 0 < lib.pygho_layer_norm_act_bwd_workspace(10, 7) <= lib.pygho_layer_norm_act_bwd_workspace(10 ** 9, 7) == 1024 * 16 * 4


def test_linear_refusals(lib):
    def fwd(y=ONE, z=ONE, x=ONE, x_ld=128, w=ONE, bdt=BF16, bias=None, norm=0, eps=1e-5, r_ld=0, r=None, m=5, k=128, n=64, act=2, dt=BF16):
        return lib.pygho_linear_act(y, z, x, x_ld, w, 128, bias, bdt, norm, None, None, BF16, eps, r, r_ld, m, k, n, act, dt, None)
    assert fwd(m=0) == 0
    assert fwd(m=-1) == 1 and fwd(k=0) == 1 and fwd(n=0) == 1 and fwd(act=4) == 1 and fwd(eps=-1.0) == 1
    assert fwd(y=None) == 1 and fwd(x=None) == 1 and fwd(w=None) == 1 and b"null" in lib.pygho_last_error()
    assert fwd(dt=F64) == 2 and fwd(bias=ONE, bdt=F16) == 2
    assert fwd(x_ld=-1) == 2 and fwd(x_ld=1 << 28) == 2 and fwd(r=ONE, r_ld=1 << 27) == 2 and b"strides" in lib.pygho_last_error()
    assert fwd(x_ld=1 << 26) == 2 and fwd(r=ONE, r_ld=1 << 26) == 2      # 32 rows of 2^27 bytes pass a 32-bit offset
    # a norm over more channels than a workgroup holds needs the pre-activation's buffer
    assert lib.pygho_linear_act_keeps(512, 512, 1, 2, BF16) == 2 and fwd(z=None, norm=1, k=512, n=512) == 1 and b"keeps" in lib.pygho_last_error()
    assert lib.pygho_linear_act_keeps(512, 512, 0, 2, BF16) == 1 and lib.pygho_linear_act_keeps(512, 512, 0, 0, BF16) == 0
    assert lib.pygho_linear_act_keeps(128, 128, 1, 2, BF16) == 0 and lib.pygho_linear_act_keeps(0, 5, 1, 2, BF16) == 0

    def bwd(gx=ONE, gw=ONE, gw_dt=BF16, gg=None, z=None, x=ONE, gy=ONE, norm=0, m=5, k=128, n=64, ws=ONE, nbytes=1 << 40):
        return lib.pygho_linear_act_bwd(gx, gw, gw_dt, None, 0, gg, BF16, None, 0, z, x, 128, ONE, 128, None, 0, norm, None, None, BF16, 1e-5, gy, 64, m,
                                        None, k, n, 2, BF16, ws, nbytes, None)
    assert bwd(gw_dt=F64) == 2 and bwd(gg=ONE) == 2 and bwd(x=None) == 1 and bwd(gy=None) == 1 and bwd(ws=None) == 1
    assert bwd(nbytes=64) == 1 and b"workspace" in lib.pygho_last_error()
    assert bwd(k=512, n=512) == 1 and b"missing" in lib.pygho_last_error()
    assert lib.pygho_linear_act_bwd_workspace(0, 4, 4, 0, 0, BF16) == 0 and lib.pygho_linear_act_bwd_workspace(5, 4, 4, 1, 2, BF16) > 0


def test_python_entries_refuse_cpu_tensors():
    from pygho_amd import _ops
    x, w = torch.randn(4, 8), torch.randn(5, 8)
    for call in (lambda: _ops.layer_norm_act(x), lambda: _ops.linear_act(x, w), lambda: _ops.linear_norm_act(x, w)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


def test_fused_mlp_on_the_cpu_is_the_stock_one():
    """the flag changes nothing where there is no device: same modules, same state_dict, same result"""
    from pygho_amd.honn.utils import MLP
    torch.manual_seed(0)
    a, b = MLP(8, 8, 2, True, norm="ln", act="silu"), MLP(8, 8, 2, True, norm="ln", act="silu", fused=True)
    assert list(a.state_dict()) == list(b.state_dict())
    b.load_state_dict(a.state_dict())
    x = torch.randn(5, 8)
    assert torch.equal(a(x, residual=x), b(x, residual=x))
