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
