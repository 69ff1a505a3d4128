"""CPU checks of the row-wise MLP operators' corners (tests/test_gpu_rowops_corners.py): no launch, no device."""
import pytest
import torch


def test_device_row_counts_past_32_bits_are_refused():
    """the count of a slot's rows is an int32 on the device: a capacity times inner dims beyond that is an error, not a wrapped count"""
    from pygho_amd import plans, rowops
    plans._ROW_FAMILIES[50000] = torch.tensor([7], dtype=torch.int32)
    try:
        assert int(rowops._device_rows((50000, 3, 2, 64))) == 42 and int(rowops._device_rows((50000, 64))) == 7
        assert rowops._device_rows((250, 200, 64)) is None and rowops._device_rows((50000,)) is None
        with pytest.raises(RuntimeError, match="32 bits"):
            rowops._device_rows((50000, 50000, 64))
    finally:
        del plans._ROW_FAMILIES[50000]


def test_an_mlp_pickled_before_the_flag_still_runs():
    import copy
    from pygho_amd.honn.utils import MLP
    torch.manual_seed(0)
    a = MLP(8, 8, 2, True, norm="ln", act="silu")
    b = copy.deepcopy(a)
    b.__dict__.pop("fused", None)                              # what unpickling an instance of the earlier class gives
    x = torch.randn(5, 8)
    assert torch.equal(a(x, residual=x), b(x, residual=x))


def test_a_call_asks_for_the_workspace_it_uses():
    """bytes by what a call wants and how its operands lie; never above the query for any call, and a call with less than its own is refused"""
    import ctypes
    import itertools
    from pygho_amd import build
    build.build(force=False, verbose=False)
    from pygho_amd._native import lib
    at, odd, bf16, f32 = 4096, 4098, 1, 0

    def need(m, k, n, norm, act, dt, gx=at, gw=1, gb=1, x=at, gy=at):
        return int(lib().pygho_linear_act_bwd_workspace_for(gx, gw, gb, x, k, gy, n, m, k, n, norm, act, dt))
    most = lambda *a: int(lib().pygho_linear_act_bwd_workspace(*a))      # noqa: E731
    big = (1831936, 128, 128, 1, 2, bf16)
    slab = (3 * 128 + 128 * 128) * 4                                     # one workgroup's sums and share of dW
    assert need(*big) == 512 * slab and most(*big) > 400 << 20           # the one-launch gradient against the plan for rows at odd addresses
    assert need(*big, x=odd) > 400 << 20
    assert need(*big, gw=0) <= 1024 * 3 * 128 * 4                        # frozen weights: sums only, dz stays on chip
    assert need(*big, gw=0, gx=None) <= 1024 * 3 * 128 * 4
    assert need(10 ** 6, 512, 512, 0, 0, bf16, gw=0, gb=0) == 512 * 512 * 2          # no norm, no activation: dz is gy, only W's transposed copy
    assert need(10 ** 6, 256, 128, 0, 0, f32, gw=0, gb=0) == 0
    assert need(10 ** 6, 512, 512, 0, 0, bf16, gw=0, gx=None) < need(10 ** 6, 512, 512, 0, 0, bf16, gb=0, gx=None) // 4
    assert need(0, 128, 128, 1, 2, bf16) == 0
    for m, (k, n), norm, act, dt in itertools.product((1, 100, 10 ** 5), ((128, 128), (100, 36), (384, 128), (256, 256), (512, 512), (20, 300)), (0, 1), (0, 2), (bf16, f32)):
        full = most(m, k, n, norm, act, dt)
        for gx, gw, gb, x in itertools.product((None, at, odd), (0, 1), (0, 1), (at, odd)):
            assert need(m, k, n, norm, act, dt, gx=gx, gw=gw, gb=gb, x=x) <= full
    one = ctypes.c_void_p(16)                                            # never dereferenced: the check fails first
    rc = lib().pygho_linear_act_bwd(one, one, bf16, None, 0, None, 0, None, 0, None, one, 128, one, 128, None, 0, 1, None, None, bf16, 1e-5, one, 128, 5000,
                                    None, 128, 128, 2, bf16, one, need(5000, 128, 128, 1, 2, bf16) - 1, None)
    assert rc == 1 and b"workspace" in lib().pygho_last_error()
    rc = lib().pygho_linear_act_bwd(one, None, 0, None, 0, None, 0, None, 0, None, one, 128, one, 128, None, 0, 1, None, None, bf16, 1e-5, one, 128, 5000,
                                    None, 128, 128, 2, bf16, None, 0, None)
    assert rc == 1 and b"null" in lib().pygho_last_error()


def test_the_flag_of_an_f32_pre_activation_leaves_the_checks_as_they_are():
    import ctypes
    from pygho_amd._native import lib
    one = ctypes.c_void_p(16)                                            # never dereferenced: the checks fail first

    def fwd(act, m=5, dt=1):
        return lib().pygho_linear_act(one, one, one, 64, one, 64, None, 0, 0, None, None, 1, 0.0, None, 0, m, 64, 64, act, dt, None)
    assert fwd(0x102, m=0) == 0 and fwd(0x104) == 1 and fwd(0x200) == 1 and fwd(0x102, dt=3) == 2
    rc = lib().pygho_linear_act_bwd(one, None, 0, None, 0, None, 0, None, 0, None, one, 512, one, 512, None, 0, 0, None, None, 1, 0.0, one, 512, 5, None, 512, 512,
                                    0x102, 1, one, 1 << 30, None)
    assert rc == 1 and b"missing" in lib().pygho_last_error()
