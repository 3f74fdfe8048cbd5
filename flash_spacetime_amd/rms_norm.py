"""Root-mean-square norm of token rows, with the residual sum before it, padded
batches, and an output in 8 bits.

The norm without a mean and a bias that a block may run in layer norm's place
(`norm.py`), as HIP kernels behind the C ABI (`fst_rms_norm_forward`,
`fst_rms_norm_backward`, `fst_rms_norm_fp8`): one pass over memory in each
direction, statistics and sums in float32, the weight's gradient summed in a fixed
order. No reference counterpart.
"""

from __future__ import annotations

from typing import Any, Optional, Tuple, Union

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _lib
from .norm import BLOCK_DTYPES, PLAIN, autocast_dtype, batch_of_rows, check_rows, token_rows


class _RmsNorm(torch.autograd.Function):
    """Fused forward and deterministic backward; keeps the normalised rows (x,
    or the residual sum it returned) and a float a row."""

    @staticmethod
    def forward(ctx: Any, x, residual, weight, eps, seqlens):  # type: ignore[override]
        dtype = BLOCK_DTYPES[x.dtype]
        b, length, lens = batch_of_rows(x, seqlens)
        n = x.shape[-1]
        param_dtype = dtype if weight is None else BLOCK_DTYPES[weight.dtype]
        w = None if weight is None else weight.contiguous()
        xr, x_stride = token_rows(x)
        rr, r_stride = (None, 0) if residual is None else token_rows(residual)
        y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
        s = None if residual is None else torch.empty_like(y)
        keep = any(ctx.needs_input_grad)
        rstd = torch.empty(b * length, device=x.device, dtype=torch.float32) if keep else None
        P = _lib.ptr
        with torch.cuda.device(x.device):
            rc = _lib.load().fst_rms_norm_forward(
                dtype, param_dtype, b, length, n, P(xr), x_stride, P(rr), r_stride, P(w), P(lens), eps,
                P(y), P(s), P(rstd), _lib.stream_handle(x.device))
        _lib.check(rc, "flash_rms_norm")
        if keep:
            ctx.save_for_backward(xr if s is None else s, w, lens, rstd)
            ctx.meta = (dtype, param_dtype, b, length, n, x_stride if s is None else n, x.shape,
                        None if weight is None else weight.dtype)
        ctx.set_materialize_grads(False)
        return y if s is None else (y, s)

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, dy: Optional[Tensor], ds: Optional[Tensor] = None):  # type: ignore[override]
        s, w, lens, rstd = ctx.saved_tensors
        dtype, param_dtype, b, length, n, s_stride, shape, w_dtype = ctx.meta
        if dy is None and ds is None:
            return (None,) * 5
        _lib.refuse_fx_recording()
        need_x, need_r, need_w = ctx.needs_input_grad[:3]
        dev = s.device
        dyr, dy_stride = token_rows(torch.zeros(shape, device=dev, dtype=s.dtype) if dy is None else dy.to(s.dtype))
        dsr, ds_stride = (None, 0) if ds is None else token_rows(ds.to(s.dtype))
        dx = torch.empty(shape, device=dev, dtype=s.dtype) if need_x or need_r else None
        dw = torch.empty(n, device=dev, dtype=w_dtype) if need_w else None
        lib = _lib.load()
        nbytes = lib.fst_rms_norm_backward_workspace_bytes(dtype, b, length, n) if need_w else 0
        ws = torch.empty(max(nbytes, 1), device=dev, dtype=torch.uint8)
        P = _lib.ptr
        with torch.cuda.device(dev):
            rc = lib.fst_rms_norm_backward(
                dtype, param_dtype, b, length, n, P(s), s_stride, P(w), P(lens), P(rstd), P(dyr), dy_stride,
                P(dsr), ds_stride, P(dx), P(dw), P(ws), nbytes, _lib.stream_handle(dev))
        _lib.check(rc, "flash_rms_norm backward")
        return dx if need_x else None, dx if need_r else None, dw, None, None


class _RmsNormFp8(torch.autograd.Function):
    """An autograd function for its records and refusals: torch's tracer takes it as a
    call, and forward-mode derivatives are refused."""

    @staticmethod
    def forward(ctx: Any, x, residual, weight, eps, seqlens):  # type: ignore[override]
        dtype = BLOCK_DTYPES[x.dtype]
        b, length, lens = batch_of_rows(x, seqlens)
        w = None if weight is None else weight.contiguous()
        xr, x_stride = token_rows(x)
        rr, r_stride = (None, 0) if residual is None else token_rows(residual)
        q = torch.empty(x.shape, device=x.device, dtype=torch.float8_e4m3fn)
        scale = torch.empty(x.shape[:-1], device=x.device, dtype=torch.float32)
        s = None if residual is None else torch.empty(x.shape, device=x.device, dtype=x.dtype)
        P = _lib.ptr
        with torch.cuda.device(x.device):
            rc = _lib.load().fst_rms_norm_fp8(
                dtype, dtype if w is None else BLOCK_DTYPES[w.dtype], b, length, x.shape[-1], P(xr), x_stride, P(rr),
                r_stride, P(w), P(lens), eps, P(q), P(scale), P(s), _lib.stream_handle(x.device))
        _lib.check(rc, "flash_rms_norm_fp8")
        outs = (q, scale) if s is None else (q, scale, s)
        ctx.mark_non_differentiable(*outs)
        return outs


def _checked(x, weight, eps, residual, seqlens):
    """The operands, in one type under autocast, once they are ones the norm takes."""
    check_rows(x, residual, weight, seqlens if seqlens is not None and seqlens.is_cuda else None)
    if autocast_dtype() is not None and all(t is None or t.dtype in BLOCK_DTYPES for t in (residual, weight)):
        wide = x.dtype if residual is None else torch.promote_types(x.dtype, residual.dtype)
        x, residual = x.to(wide), None if residual is None else residual.to(wide)
        if weight is not None and weight.dtype not in (wide, torch.float32):
            weight = weight.float()
    n = x.shape[-1]
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"residual must have x's shape and dtype ({tuple(x.shape)}, {x.dtype}), got "
                         f"{tuple(residual.shape)}, {residual.dtype}")
    if weight is not None and weight.shape != (n,):
        raise ValueError(f"weight must be [N={n}], got {tuple(weight.shape)}")
    if weight is not None and weight.dtype not in (x.dtype, torch.float32):
        raise ValueError(f"weight must be {x.dtype} or float32, got {weight.dtype}")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    return x, weight, residual


def flash_rms_norm(
    x: Tensor,
    weight: Optional[Tensor] = None,
    eps: float = 1e-6,
    *,
    residual: Optional[Tensor] = None,
    seqlens: Optional[Tensor] = None,
) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    """Root-mean-square norm over the last dimension of `x [.., N]` (bfloat16, float16
    or float32; N up to 16384): `x / sqrt(mean(x^2) + eps) * weight`.

    `weight` `[N]` may be omitted; it is of x's dtype or float32, and gets a gradient
    of its own. `residual`, `seqlens`, autocast and strides are `flash_layer_norm`'s:
    with `residual` the norm is of `s = x + residual`, rounded to x's dtype, and
    `(y, s)` is returned; with `seqlens` rows past an event's length are not read and come
    back as zeros everywhere. A row whose squares overflow float32 (values past 1e19)
    comes out as zeros, and with eps = 0 one whose squares all vanish (below 1e-23) is not
    finite.

    Statistics and sums are float32; results are bitwise reproducible.
    """
    if x.is_cuda and all(t is None or type(t) in PLAIN for t in (x, residual, weight, seqlens)):
        host = _lib.host()
        out = None if host is None else host.rms_norm(x, residual, weight, eps, seqlens)
        if out is not None:
            return out
    x, weight, residual = _checked(x, weight, eps, residual, seqlens)
    return _RmsNorm.apply(x, residual, weight, float(eps), seqlens)


def flash_rms_norm_fp8(
    x: Tensor,
    weight: Optional[Tensor] = None,
    eps: float = 1e-6,
    *,
    residual: Optional[Tensor] = None,
    seqlens: Optional[Tensor] = None,
) -> Union[Tuple[Tensor, Tensor], Tuple[Tensor, Tensor, Tensor]]:
    """`flash_rms_norm` with its output in 8 bits and one scale a row, for products in
    8 bits: `(q, scale)`, or `(q, scale, s)` with `residual`.

    `q` is x's shape in torch.float8_e4m3fn, `scale` float32 of the shape without the
    last dimension, and `q * scale` the normalised row: the row's largest value stands
    at 448, the type's largest. The scale is at least 2^-126, so that of a row of zeros
    is not 0; padding rows are zeros with scale 0. q is rounded once, from the
    float32 row. It has no derivative: operands that ask for one are refused where
    gradients are recorded.
    """
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual)):
        raise ValueError("flash_rms_norm_fp8 has no derivative: call it under torch.no_grad(), or on detached tensors")
    if x.is_cuda and all(t is None or type(t) in PLAIN for t in (x, residual, weight, seqlens)):
        host = _lib.host()
        out = None if host is None else host.rms_norm_fp8(x, residual, weight, eps, seqlens)
        if out is not None:
            return out
    x, weight, residual = _checked(x, weight, eps, residual, seqlens)
    return _RmsNormFp8.apply(x, residual, weight, float(eps), seqlens)
