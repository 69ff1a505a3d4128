"""
Row-wise MLP blocks without a batch norm (reference honn/utils.py:64-142: LayerNorm, the activations, MLP) as single operators:

    layer_norm_act(x, g, h, eps, act, residual)          act(LayerNorm(x) * g + h) + residual

over the last dim of x, any leading dims.  f32 / bf16 / f16; statistics and sums in f32, every output rounded once.  Parameters may be
stored in x's dtype or (master weights) in f32; their gradients come back in their own dtype.  Gradients are first order only.
"""
from __future__ import annotations

from ctypes import byref, c_int
from typing import Optional, Tuple

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from ._native import DTYPE_CODE, check, lib, ptr, require_device, stream_ptr

from .plans import dyn_rows

ROW_ACT_CODE = {"none": 0, "relu": 1, "silu": 2, "elu": 3}      # enum pygho_row_act
_ROW_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def _row_args(x: Tensor, act: str, what: str) -> None:
    if act not in ROW_ACT_CODE:
        raise ValueError(f"pygho_amd.{what}: activation {act!r} is not one of {sorted(ROW_ACT_CODE)}")
    if not isinstance(x, Tensor) or x.dim() < 1:
        raise ValueError(f"pygho_amd.{what}: x must be a tensor with at least one dim")
    if x.dtype not in _ROW_DTYPES:
        raise TypeError(f"pygho_amd.{what}: {x.dtype} rows (f32, bf16 or f16)")
    if x.shape[-1] < 1:
        raise ValueError(f"pygho_amd.{what}: rows without channels")


def _row_operand(t: Optional[Tensor], shape, dtypes, name: str, what: str) -> None:
    if t is None:
        return
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"pygho_amd.{what}: {name} has shape {tuple(t.shape)}, needs {tuple(shape)}")
    if t.dtype not in dtypes:
        raise TypeError(f"pygho_amd.{what}: {name} is {t.dtype}, needs {' or '.join(str(d) for d in dtypes)}")


def _rows(t: Optional[Tensor], c: int) -> Tuple[Optional[Tensor], int]:
    """(rows, width) view of t and its row stride in elements; a copy only where the channels of a row are not adjacent"""
    if t is None:
        return None, 0
    t2 = t if t.dim() == 2 else t.reshape(-1, c)
    if c > 1 and t2.stride(1) != 1:
        t2 = t2.contiguous()
    return t2, (t2.stride(0) if t2.shape[0] > 1 else c)


def _norm_params(x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor]):
    """weight / bias as the kernels take them: contiguous, both in x's dtype or both in f32"""
    have = [p for p in (weight, bias) if p is not None]
    if all(p.dtype == x.dtype for p in have):
        dt = x.dtype
    else:
        dt = torch.float32
    w, b = (None if p is None else p.detach().to(dt).contiguous() for p in (weight, bias))
    return w, b, DTYPE_CODE[dt]


def _layer_norm_fwd(x: Tensor, w, b, pdt: int, eps: float, act: str, residual: Optional[Tensor], out_shape, dtype: torch.dtype) -> Tensor:
    c = x.shape[-1]
    x2, x_ld = _rows(x, c)
    r2, r_ld = _rows(residual, c)
    y = torch.empty(out_shape, dtype=dtype, device=x.device)
    check(lib().pygho_layer_norm_act(ptr(y), ptr(x2), x_ld, ptr(w), ptr(b), pdt, ptr(r2), r_ld, x2.shape[0], c, float(eps), ROW_ACT_CODE[act],
                                     DTYPE_CODE[dtype], DTYPE_CODE[x2.dtype], stream_ptr(x.device)), "layer_norm_act")
    return y


def fold_partials(slabs: Tensor, n_slabs: int, stride: int, outs) -> None:
    """add the columns of the first n_slabs f32 slabs into `outs`: up to four (tensor or None, length)"""
    args = []
    for k in range(4):
        t, n = outs[k] if k < len(outs) else (None, 0)
        args += [ptr(t), n, 0 if t is None else DTYPE_CODE[t.dtype]]
    check(lib().pygho_fold_partials(*args, ptr(slabs), n_slabs, stride, stream_ptr(slabs.device)), "fold_partials")


def _layer_norm_bwd(x: Tensor, gy: Tensor, w, b, pdt: int, eps: float, act: str, out_dtypes, want_colsum: bool = False):
    """(gx (rows, c) in gy's dtype, gradients of weight, bias and the column sums of gx in `out_dtypes`; None where that is None)"""
    c = x.shape[-1]
    x2, x_ld = _rows(x, c)
    gy2, gy_ld = _rows(gy, c)
    m, dev = x2.shape[0], x2.device
    sums = 3 if want_colsum else 2
    stride = (sums * c + 3) // 4 * 4
    gx = torch.empty((m, c), dtype=gy2.dtype, device=dev)
    slabs = torch.empty((max(1, int(lib().pygho_layer_norm_act_bwd_slabs(m))), stride), dtype=torch.float32, device=dev)
    n = c_int(0)
    check(lib().pygho_layer_norm_act_bwd(ptr(gx), ptr(slabs), stride, sums, byref(n), ptr(x2), x_ld, ptr(gy2), gy_ld, ptr(w), ptr(b), pdt, m,
                                         ptr(dyn_rows(m)), c, float(eps), ROW_ACT_CODE[act], DTYPE_CODE[gy2.dtype], DTYPE_CODE[x2.dtype],
                                         stream_ptr(dev)), "layer_norm_act_bwd")
    outs = [None if d is None else torch.empty(c, dtype=d, device=dev) for d in out_dtypes]
    if any(o is not None for o in outs):
        fold_partials(slabs, n.value, stride, [(o, c) for o in outs[:sums]])
    return (gx,) + tuple(outs)


class _LayerNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, eps, act):
        w, b, pdt = _norm_params(x, weight, bias)
        xs = x if x.dim() == 2 and (x.stride(1) == 1 or x.shape[1] == 1) else _rows(x, x.shape[-1])[0]
        y = _layer_norm_fwd(xs, w, b, pdt, eps, act, residual, x.shape, x.dtype)
        ctx.save_for_backward(xs, w, b)
        ctx.meta = (pdt, eps, act, x.shape, None if weight is None else weight.dtype, None if bias is None else bias.dtype)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        xs, w, b = ctx.saved_tensors
        pdt, eps, act, shape, w_dtype, b_dtype = ctx.meta
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        gx = gw = gb = None
        if need_x or need_w or need_b:
            gx, gw, gb = _layer_norm_bwd(xs, gy, w, b, pdt, eps, act, (w_dtype if need_w else None, b_dtype if need_b else None))
            gx = gx.view(shape) if need_x else None
        return gx, gw, gb, (gy if need_r else None), None, None


def layer_norm_act(x: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None, eps: float = 1e-5, act: str = "none",
                   residual: Optional[Tensor] = None) -> Tensor:
    """act(LayerNorm(x) * weight + bias) + residual over the last dim (biased variance, ``torch.nn.LayerNorm``'s formula); act is one of
    "none", "relu", "silu", "elu".  weight / bias: (C,) in x's dtype or f32, residual: x's shape and dtype.  One launch forward, two
    backward (rows and gradients of the parameters; a second that adds the workgroups' shares in a fixed order)."""
    what = "layer_norm_act"
    _row_args(x, act, what)
    c = x.shape[-1]
    _row_operand(weight, (c,), _ROW_DTYPES, "weight", what)
    _row_operand(bias, (c,), _ROW_DTYPES, "bias", what)
    _row_operand(residual, x.shape, (x.dtype,), "residual", what)
    if not eps >= 0:
        raise ValueError(f"pygho_amd.{what}: eps must not be negative")
    require_device(x, weight, bias, residual)
    return _LayerNormAct.apply(x, weight, bias, residual, eps, act)
