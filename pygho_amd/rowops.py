"""
Row-wise MLP blocks without a batch norm (reference honn/utils.py:64-142: LayerNorm, the activations, MLP) as single operators:

    layer_norm_act(x, g, h, eps, act, residual)             act(LayerNorm(x) * g + h) + residual
    linear_act(x, W, b, act, residual)                      act(x W^T + b) + residual
    linear_norm_act(x, W, b, g, h, eps, act, residual)      act(LayerNorm(x W^T + b) * g + h) + residual

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


def _linear_fwd(x2: Tensor, x_ld: int, w: Tensor, w_ld: int, b, bdt: int, norm, eps: float, act: str, residual: Optional[Tensor], out_shape,
                out_dtype: torch.dtype) -> Tensor:
    """norm: None, or (g, h, dtype code)"""
    n, k = w.shape
    r2, r_ld = _rows(residual, n)
    y = torch.empty(out_shape, dtype=out_dtype, device=x2.device)
    g, h, pdt = norm if norm is not None else (None, None, 0)
    check(lib().pygho_linear_act(ptr(y), ptr(x2), x_ld, ptr(w), w_ld, ptr(b), bdt, 0 if norm is None else 1, ptr(g), ptr(h), pdt, float(eps),
                                 ptr(r2), r_ld, x2.shape[0], k, n, ROW_ACT_CODE[act], DTYPE_CODE[x2.dtype], DTYPE_CODE[out_dtype],
                                 stream_ptr(x2.device)), "linear_act")
    return y


class _LinearAct(torch.autograd.Function):
    """act([LayerNorm](x W^T + b) [* g + h]) + residual.  What backward reads: x and the parameters; the product itself is formed again, except
    behind a norm over more channels than one workgroup holds (pygho_linear_norm_max), where it is kept in f32."""

    @staticmethod
    def forward(ctx, x, weight, bias, g, h, residual, eps, act, normed):
        from .blocks import param_as
        dt = x.dtype
        n, k = weight.shape
        w, w_ld = _matrix(param_as(weight, dt).detach())
        b, bdt = _bias(bias, dt)
        x2, x_ld = _rows(x, k)
        norm = None
        if normed:
            norm = _norm_params(x, g, h)
        out_shape = tuple(x.shape[:-1]) + (n,)
        z = None
        if normed and n > int(lib().pygho_linear_norm_max()):
            z = _linear_fwd(x2, x_ld, w, w_ld, b, bdt, None, 0.0, "none", None, (x2.shape[0], n), torch.float32)
            y = _layer_norm_fwd(z, norm[0], norm[1], norm[2], eps, act, residual, out_shape, dt)
        else:
            y = _linear_fwd(x2, x_ld, w, w_ld, b, bdt, norm, eps, act, residual, out_shape, dt)
        ctx.save_for_backward(x2, w, b, z, *(norm[:2] if normed else (None, None)))
        ctx.meta = (bdt, norm[2] if normed else 0, eps, act, normed, x.shape, weight.dtype,
                    *(None if t is None else t.dtype for t in (bias, g, h)))
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        x2, w, b, z, g, h = ctx.saved_tensors
        bdt, pdt, eps, act, normed, x_shape, w_dtype, b_dtype, g_dtype, h_dtype = ctx.meta
        need_x, need_w, need_b, need_g, need_h, need_r = ctx.needs_input_grad[:6]
        out = [None] * 6
        out[5] = gy if need_r else None
        if not (need_x or need_w or need_b or need_g or need_h):
            return (*out, None, None, None)
        n, k = w.shape
        w, w_ld = _matrix(w)
        x2, x_ld = _rows(x2, k)
        gy2, gy_ld = _rows(gy, n)
        m, dev, dt = x2.shape[0], x2.device, x2.dtype
        st, code, m_dev = stream_ptr(dev), DTYPE_CODE[dt], dyn_rows(m)
        if z is not None:
            dz, out[3], out[4], out[2] = _layer_norm_bwd(z, gy2, g, h, pdt, eps, act, (g_dtype if need_g else None, h_dtype if need_h else None,
                                                                                       b_dtype if need_b else None), want_colsum=True)
            dz_ld = n
        elif act == "none" and not normed:
            dz, dz_ld = gy2, gy_ld
        else:
            dz, dz_ld = torch.empty((m, n), dtype=dt, device=dev), n
            stride = (2 * n + 3) // 4 * 4
            slabs = torch.empty((max(1, int(lib().pygho_linear_act_dz_slabs(m))), stride), dtype=torch.float32, device=dev) if normed else None
            used = c_int(0)
            check(lib().pygho_linear_act_dz(ptr(dz), ptr(slabs), stride, byref(used), ptr(x2), x_ld, ptr(w), w_ld, ptr(b), bdt, 1 if normed else 0,
                                            ptr(g), ptr(h), pdt, float(eps), ptr(gy2), gy_ld, m, ptr(m_dev), k, n, ROW_ACT_CODE[act], code, st),
                  "linear_act_dz")
            if need_g or need_h:
                out[3] = torch.empty(n, dtype=g_dtype, device=dev) if need_g else None
                out[4] = torch.empty(n, dtype=h_dtype, device=dev) if need_h else None
                fold_partials(slabs, used.value, stride, [(out[3], n), (out[4], n)])
        if need_x:
            gx = torch.empty((m, k), dtype=dt, device=dev)
            check(lib().pygho_linear_dx(ptr(gx), ptr(dz), dz_ld, ptr(w), w_ld, m, k, n, code, st), "linear_dx")
            out[0] = gx.view(x_shape)
        if need_w or (need_b and out[2] is None):
            colsum = need_b and out[2] is None
            count = int(lib().pygho_linear_dw_slabs(m, k, n))
            stride = (n * k + (n if colsum else 0) + 3) // 4 * 4
            slabs = torch.empty((max(1, count), stride), dtype=torch.float32, device=dev)
            check(lib().pygho_linear_dw(ptr(slabs), stride, ptr(dz), dz_ld, ptr(x2), x_ld, m, ptr(m_dev), k, n, 1 if colsum else 0, code, st),
                  "linear_dw")
            out[1] = torch.empty((n, k), dtype=w_dtype, device=dev) if need_w else None
            if colsum:
                out[2] = torch.empty(n, dtype=b_dtype, device=dev)
            fold_partials(slabs, count, stride, [(out[1], n * k), (out[2] if colsum else None, n if colsum else 0)])
        return (*out, None, None, None)


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
    bias (N,): in x's dtype, or f32 master parameters (the product then takes their copy in x's dtype, `param_as`), residual: the output's
    shape and x's dtype.  Backward: the gradient of the pre-activation (formed again from x), dX and dW / db on the same tiled product."""
    _linear_args(x, weight, bias, act, residual, "linear_act")
    return _LinearAct.apply(x, weight, bias, None, None, residual, 0.0, act, False)


def linear_norm_act(x: Tensor, weight: Tensor, bias: Optional[Tensor] = None, norm_weight: Optional[Tensor] = None,
                    norm_bias: Optional[Tensor] = None, eps: float = 1e-5, act: str = "none", residual: Optional[Tensor] = None) -> Tensor:
    """act(LayerNorm(x @ weight^T + bias) * norm_weight + norm_bias) + residual: one [Linear, LayerNorm, act] block of an MLP with the layer's
    residual connection.  Up to 256 output channels in one launch (the pre-activation never reaches memory), beyond that the product in f32
    and `layer_norm_act` over it.  Arguments as in `linear_act` and `layer_norm_act`."""
    what = "linear_norm_act"
    _linear_args(x, weight, bias, act, residual, what)
    n = weight.shape[0]
    _row_operand(norm_weight, (n,), _ROW_DTYPES, "norm_weight", what)
    _row_operand(norm_bias, (n,), _ROW_DTYPES, "norm_bias", what)
    if not eps >= 0:
        raise ValueError(f"pygho_amd.{what}: eps must not be negative")
    require_device(x, norm_weight, norm_bias)
    return _LinearAct.apply(x, weight, bias, norm_weight, norm_bias, residual, eps, act, True)
