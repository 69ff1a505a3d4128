"""
Row-wise MLP blocks without a batch norm (reference honn/utils.py:64-142: LayerNorm, the activations, MLP) as single operators:

    layer_norm_act(x, g, h, eps, act, residual)             act(LayerNorm(x) * g + h) + residual
    linear_act(x, W, b, act, residual)                      act(x W^T + b) + residual
    linear_norm_act(x, W, b, g, h, eps, act, residual)      act(LayerNorm(x W^T + b) * g + h) + residual

over the last dim of x, any leading dims.  f32 / bf16 / f16; statistics and sums in f32, every output rounded once.  With 16-bit rows the gradient
of x W^T + b enters the two products of the backward (x's and W's gradient) rounded to the rows' type, as the matrix cores take it; the gradients of
bias and norm are sums of its f32 values.  Parameters may be stored in x's dtype or (master weights) in f32; their gradients come back in their own
dtype.  Gradients are first order only.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from ._native import DTYPE_CODE, check, lib, ptr, require_device, stream_ptr

from .blocks import param_as
from .plans import dyn_rows

ROW_ACT_CODE = {"none": 0, "relu": 1, "silu": 2, "elu": 3}      # enum pygho_row_act
_Z_F32 = 0x100                                                   # PYGHO_ROW_Z_F32
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


def _rows(t: Optional[Tensor], c: int, within: int = 0) -> Tuple[Optional[Tensor], int]:
    """(rows, width) view of t and its row stride in elements; a copy where the channels of a row are not adjacent, where the leading dims do
    not merge into one stride, and where the rows are `within` bytes or more apart (0: any distance)"""
    if t is None:
        return None, 0
    t2 = t if t.dim() == 2 else t.reshape(-1, c)
    if (c > 1 and t2.stride(1) != 1) or (within and t2.shape[0] > 1 and t2.stride(0) * t2.element_size() >= within):
        t2 = t2.contiguous()
    return t2, (t2.stride(0) if t2.shape[0] > 1 else c)


def _device_rows(shape) -> Optional[Tensor]:
    """the device-side count of the rows of a (.., C) tensor inside a batch slot (None: all rows are true ones).  As everywhere the extent of
    dim 0 names the row family (`plans.row_families`); dims between it and the channels multiply its count"""
    count = dyn_rows(shape[0]) if len(shape) > 1 else None
    inner = math.prod(shape[1:-1])
    if count is None or inner == 1:
        return count
    if shape[0] * inner > 2 ** 31 - 1:
        raise RuntimeError(f"pygho_amd: {shape[0]} x {inner} rows of a batch slot pass the device-side row count's 32 bits")
    return count[:1] * inner


def _norm_params(x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor]):
    """weight / bias as the kernels take them: contiguous, both in x's dtype or both in f32"""
    have = [p for p in (weight, bias) if p is not None]
    if all(p.dtype == x.dtype for p in have):
        dt = x.dtype
    else:
        dt = torch.float32
    w, b = (None if p is None else p.detach().to(dt).contiguous() for p in (weight, bias))
    return w, b, DTYPE_CODE[dt]


def _workspace(nbytes: int, dev) -> Optional[Tensor]:
    return torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None


def _grad(need: bool, shape, dtype, dev):
    """(tensor or None, address, dtype code) of a parameter's gradient"""
    if not need:
        return None, None, 0
    t = torch.empty(shape, dtype=dtype, device=dev)
    return t, t.data_ptr(), DTYPE_CODE[dtype]


class _LayerNormAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, eps, act):
        w, b, pdt = _norm_params(x, weight, bias)
        c = x.shape[-1]
        x2, x_ld = _rows(x, c)
        r2, r_ld = _rows(residual, c)
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        check(lib().pygho_layer_norm_act(ptr(y), ptr(x2), x_ld, ptr(w), ptr(b), pdt, ptr(r2), r_ld, x2.shape[0], c, float(eps), ROW_ACT_CODE[act],
                                         DTYPE_CODE[x.dtype], stream_ptr(x.device)), "layer_norm_act")
        ctx.save_for_backward(x2, w, b)
        ctx.meta = (x_ld, pdt, eps, act, x.shape, None if weight is None else weight.dtype, None if bias is None else bias.dtype)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        if not (need_x or need_w or need_b):
            return None, None, None, (gy if need_r else None), None, None
        x2, w, b = ctx.saved_tensors
        x_ld, pdt, eps, act, shape, w_dtype, b_dtype = ctx.meta
        (m, c), dev, code = x2.shape, x2.device, DTYPE_CODE[x2.dtype]
        gy2, gy_ld = _rows(gy, c)
        gx = torch.empty(shape, dtype=x2.dtype, device=dev)
        gw, gw_ptr, gw_code = _grad(need_w, c, w_dtype, dev)
        gb, gb_ptr, gb_code = _grad(need_b, c, b_dtype, dev)
        nbytes = int(lib().pygho_layer_norm_act_bwd_workspace(m, c))
        ws, count = _workspace(nbytes, dev), _device_rows(shape)
        check(lib().pygho_layer_norm_act_bwd(ptr(gx), gw_ptr, gw_code, gb_ptr, gb_code, ptr(x2), x_ld, ptr(gy2), gy_ld, ptr(w), ptr(b), pdt, m,
                                             ptr(count), c, float(eps), ROW_ACT_CODE[act], code, ptr(ws), nbytes, stream_ptr(dev)),
              "layer_norm_act_bwd")
        return (gx if need_x else None), gw, gb, (gy if need_r else None), None, None


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


# ---- linear maps ----------------------------------------------------------------------------------------------------------------------
def _matrix(w: Tensor) -> Tuple[Tensor, int]:
    """a (n, k) weight with adjacent k and its row stride"""
    if w.shape[1] > 1 and w.stride(1) != 1:
        w = w.contiguous()
    return w, (w.stride(0) if w.shape[0] > 1 else w.shape[1])


def _bias(b: Optional[Tensor], dtype: torch.dtype):
    if b is None:
        return None, 0
    b = b.detach()
    if b.dtype not in (dtype, torch.float32):
        b = b.float()
    return b.contiguous(), DTYPE_CODE[b.dtype]


class _LinearAct(torch.autograd.Function):
    """act([LayerNorm](x W^T + b) [* g + h]) + residual.  Kept for backward: x, the parameters and, where the C side says so
    (pygho_linear_act_keeps: W does not fit a CU's LDS), the pre-activation."""

    @staticmethod
    def forward(ctx, x, weight, bias, g, h, residual, eps, act, normed, training):
        dt, dev = x.dtype, x.device
        n, k = weight.shape
        w, w_ld = _matrix(param_as(weight, dt).detach())
        b, bdt = _bias(bias, dt)
        x2, x_ld = _rows(x, k)
        r2, r_ld = _rows(residual, n)
        gg, hh, pdt = _norm_params(x, g, h) if normed else (None, None, 0)
        m, code = x2.shape[0], DTYPE_CODE[dt]
        y = torch.empty(tuple(x.shape[:-1]) + (n,), dtype=dt, device=dev)
        keeps = int(lib().pygho_linear_act_keeps(k, n, int(normed), ROW_ACT_CODE[act], code))
        z = None
        # (`training`: the caller's grad mode.  In here it is always off, and needs_input_grad says what the inputs ask for in either mode)
        if keeps == 2 or (keeps == 1 and training and any(ctx.needs_input_grad[:5])):
            # in f32 for 16-bit rows too: the slope is then that of the unrounded z, as in the forms that form it again (a z rounded to bf16 moves silu's
            # slope by up to 2^-8).  Training bf16 65536 x 512 -> 512 361 us, with 16 bits 354; 300 -> 300 368, 342
            z = torch.empty((m, n), dtype=torch.float32, device=dev)
        check(lib().pygho_linear_act(ptr(y), ptr(z), ptr(x2), x_ld, ptr(w), w_ld, ptr(b), bdt, int(normed), ptr(gg), ptr(hh), pdt, float(eps),
                                     ptr(r2), r_ld, m, k, n, ROW_ACT_CODE[act] | _Z_F32, code, stream_ptr(dev)), "linear_act")
        ctx.save_for_backward(x2, w, b, z, gg, hh)
        ctx.meta = (x_ld, w_ld, bdt, pdt, eps, act, normed, x.shape, weight.dtype, *(None if t is None else t.dtype for t in (bias, g, h)))
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        need_x, need_w, need_b, need_g, need_h, need_r = ctx.needs_input_grad[:6]
        res = gy if need_r else None
        if not (need_x or need_w or need_b or need_g or need_h):
            return None, None, None, None, None, res, None, None, None, None
        x2, w, b, z, g, h = ctx.saved_tensors
        x_ld, w_ld, bdt, pdt, eps, act, normed, x_shape, w_dtype, b_dtype, g_dtype, h_dtype = ctx.meta
        n, k = w.shape
        gy2, gy_ld = _rows(gy, n, 1 << 27)                     # (the caller of a forward chose its strides, nobody chooses a gradient's)
        m, dev, code = x2.shape[0], x2.device, DTYPE_CODE[x2.dtype]
        gx = torch.empty(x_shape, dtype=x2.dtype, device=dev) if need_x else None
        gw, gw_ptr, gw_code = _grad(need_w, (n, k), w_dtype, dev)
        gb, gb_ptr, gb_code = _grad(need_b, n, b_dtype, dev)
        gg, gg_ptr, gg_code = _grad(need_g, n, g_dtype, dev)
        gh, gh_ptr, gh_code = _grad(need_h, n, h_dtype, dev)
        nbytes = int(lib().pygho_linear_act_bwd_workspace_for(ptr(gx), need_w, need_b, ptr(x2), x_ld, ptr(gy2), gy_ld, m, k, n, int(normed),
                                                              ROW_ACT_CODE[act], code))
        ws, count = _workspace(nbytes, dev), _device_rows(x_shape)
        check(lib().pygho_linear_act_bwd(ptr(gx), gw_ptr, gw_code, gb_ptr, gb_code, gg_ptr, gg_code, gh_ptr, gh_code, ptr(z), ptr(x2), x_ld, ptr(w),
                                         w_ld, ptr(b), bdt, int(normed), ptr(g), ptr(h), pdt, float(eps), ptr(gy2), gy_ld, m, ptr(count),
                                         k, n, ROW_ACT_CODE[act] | _Z_F32, code, ptr(ws), nbytes, stream_ptr(dev)), "linear_act_bwd")
        return gx, gw, gb, gg, gh, res, None, None, None, None


def _linear_args(x: Tensor, weight: Tensor, bias: Optional[Tensor], act: str, residual: Optional[Tensor], what: str) -> None:
    _row_args(x, act, what)
    if not isinstance(weight, Tensor) or weight.dim() != 2 or weight.shape[1] != x.shape[-1] or weight.shape[0] < 1:
        raise ValueError(f"pygho_amd.{what}: weight must be (out, {x.shape[-1]}) with at least one output channel")
    if weight.dtype not in (x.dtype, torch.float32):
        raise TypeError(f"pygho_amd.{what}: weight is {weight.dtype}, needs {x.dtype} or float32")
    n = weight.shape[0]
    _row_operand(bias, (n,), _ROW_DTYPES, "bias", what)
    _row_operand(residual, tuple(x.shape[:-1]) + (n,), (x.dtype,), "residual", what)
    require_device(x, weight, bias, residual)


def linear_act(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, act: str = "none", residual: Optional[Tensor] = None) -> Tensor:
    """act(x @ weight^T + bias) + residual over the last dim of x in one launch; act is one of "none", "relu", "silu", "elu".  weight (N, K) and
    bias (N,): in x's dtype, or f32 master parameters (the product then takes W's copy in x's dtype, `param_as`), residual: the output's shape and
    x's dtype.  Rows of x and residual less than 2^27 bytes apart."""
    _linear_args(x, weight, bias, act, residual, "linear_act")
    return _LinearAct.apply(x, weight, bias, None, None, residual, 0.0, act, False, torch.is_grad_enabled())


def linear_norm_act(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, norm_weight: Optional[Tensor] = None,
                    norm_bias: Optional[Tensor] = None, eps: float = 1e-5, act: str = "none", residual: Optional[Tensor] = None) -> Tensor:
    """act(LayerNorm(x @ weight^T + bias) * norm_weight + norm_bias) + residual: one [Linear, LayerNorm, act] block of an MLP with the layer's
    residual connection.  One launch where W fits a CU's LDS (up to 256 output channels; the pre-activation never reaches memory), otherwise the
    product in f32 and the norm over it.  Arguments as in `linear_act` and `layer_norm_act`."""
    what = "linear_norm_act"
    _linear_args(x, weight, bias, act, residual, what)
    n = weight.shape[0]
    _row_operand(norm_weight, (n,), _ROW_DTYPES, "norm_weight", what)
    _row_operand(norm_bias, (n,), _ROW_DTYPES, "norm_bias", what)
    if not eps >= 0:
        raise ValueError(f"pygho_amd.{what}: eps must not be negative")
    require_device(x, norm_weight, norm_bias)
    return _LinearAct.apply(x, weight, bias, norm_weight, norm_bias, residual, eps, act, True, torch.is_grad_enabled())
