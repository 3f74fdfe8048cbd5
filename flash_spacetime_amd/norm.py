"""Layer norm of token rows, with the residual sum before it and padded batches.

The norm of graphnet's `Block_rel` (the model block around the reference's
operator, reference README.md:105-116), as HIP kernels behind the C ABI
(`fst_layer_norm_forward`, `fst_layer_norm_backward`): one pass over memory in
each direction, statistics and sums in float32, the parameters' gradients
summed in a fixed order. No reference counterpart.
"""

from __future__ import annotations

from typing import Any, Optional, Tuple, Union

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _lib

BLOCK_DTYPES = {torch.bfloat16: _lib.FST_BF16, torch.float16: _lib.FST_F16, torch.float32: _lib.FST_F32}


def token_rows(t: Tensor, align: int = 1) -> Tuple[Tensor, int]:
    """`t [.., N]` as rows for the kernels: the tensor whose address and row
    stride (elements) they take, itself where its rows lie a fixed stride of at
    least N apart with their elements adjacent (start and stride multiples of
    `align` bytes), else a contiguous copy."""
    n = t.shape[-1]
    rows = t.numel() // n if n else 0
    if rows > 1:
        try:
            flat = t.view(rows, n)
            stride = flat.stride(0)
        except RuntimeError:
            return t.contiguous(), n
    else:
        flat, stride = t, n
    if (n > 1 and t.stride(-1) != 1) or stride < n:
        return t.contiguous(), n
    if t.data_ptr() % align or stride * t.element_size() % align:
        return t.clone(memory_format=torch.contiguous_format), n
    return t, stride


def batch_of_rows(x: Tensor, seqlens: Optional[Tensor]) -> Tuple[int, int, Optional[Tensor]]:
    """(B, L, int32 lengths on x's device) of a padded `x [B, L, N]`, or of rows `x
    [L, N]` with the one length [1]; or every row of `x [.., N]` as one event without
    lengths."""
    if seqlens is None:
        return 1, x.numel() // x.shape[-1], None
    if x.dim() != 3 and not (x.dim() == 2 and tuple(seqlens.shape) == (1,)):
        raise ValueError(f"seqlens needs padded x [B, L, features], or [1] packed x [T, features], got "
                         f"{tuple(x.shape)}, seqlens {tuple(seqlens.shape)}")
    batch, length = (1, *x.shape[:1]) if x.dim() == 2 else x.shape[:2]
    if seqlens.dim() != 1 or seqlens.shape[0] != batch:
        raise ValueError(f"seqlens must be [B={batch}], got {tuple(seqlens.shape)}")
    if seqlens.dtype.is_floating_point or seqlens.dtype == torch.bool:
        raise ValueError(f"seqlens must be an integer tensor, got {seqlens.dtype}")
    return batch, length, seqlens.to(device=x.device, dtype=torch.int32).contiguous()


def check_rows(x: Tensor, *others: Optional[Tensor]) -> int:
    """The C dtype of x, once x and the others are tensors of one GPU."""
    _lib.refuse_fx_recording()
    for t in (x, *others):
        if t is not None:
            _lib.require_gpu(t)
            if t.device != x.device:
                raise ValueError(f"all tensors must be on {x.device}, got one on {t.device}")
    if x.dtype not in BLOCK_DTYPES:
        raise ValueError(f"x must be bfloat16, float16 or float32, got {x.dtype}")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must be [.., features], got {tuple(x.shape)}")
    return BLOCK_DTYPES[x.dtype]


def autocast_dtype() -> Optional[torch.dtype]:
    """The type torch.autocast has the GPU's products in; None outside of it."""
    return torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else None


# Tensors without methods of their own: calls of these go through the host
# extension (csrc/fst_block_host.cpp), which gives back None for what it leaves to
# the Python path.
PLAIN = (Tensor, torch.nn.Parameter)


class _LayerNorm(torch.autograd.Function):
    """Fused forward and deterministic backward; keeps the normalised rows
    (x, or the residual sum it returned) and two floats a row."""

    @staticmethod
    def forward(ctx: Any, x, residual, weight, bias, eps, seqlens):  # type: ignore[override]
        dtype = BLOCK_DTYPES[x.dtype]
        b, length, lens = batch_of_rows(x, seqlens)
        n = x.shape[-1]
        params = [t for t in (weight, bias) if t is not None]
        param_dtype = BLOCK_DTYPES[params[0].dtype] if params else dtype
        w = None if weight is None else weight.contiguous()
        bb = None if bias is None else bias.contiguous()
        xr, x_stride = token_rows(x)
        rr, r_stride = (None, 0) if residual is None else token_rows(residual)
        y = torch.empty(x.shape, device=x.device, dtype=x.dtype)
        s = None if residual is None else torch.empty_like(y)
        keep = any(ctx.needs_input_grad)
        stats = torch.empty(b * length, 2, device=x.device, dtype=torch.float32) if keep else None
        P = _lib.ptr
        with torch.cuda.device(x.device):
            rc = _lib.load().fst_layer_norm_forward(
                dtype, param_dtype, b, length, n, P(xr), x_stride, P(rr), r_stride, P(w), P(bb), P(lens), eps,
                P(y), P(s), P(stats), _lib.stream_handle(x.device))
        _lib.check(rc, "flash_layer_norm")
        if keep:
            ctx.save_for_backward(xr if s is None else s, w, lens, stats)
            ctx.meta = (dtype, param_dtype, b, length, n, x_stride if s is None else n, x.shape,
                        None if weight is None else weight.dtype, None if bias is None else bias.dtype)
        ctx.set_materialize_grads(False)
        return y if s is None else (y, s)

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, dy: Optional[Tensor], ds: Optional[Tensor] = None):  # type: ignore[override]
        s, w, lens, stats = ctx.saved_tensors
        dtype, param_dtype, b, length, n, s_stride, shape, w_dtype, b_dtype = ctx.meta
        if dy is None and ds is None:
            return (None,) * 6
        _lib.refuse_fx_recording()
        need_x, need_r, need_w, need_b = ctx.needs_input_grad[:4]
        dev = s.device
        dyr, dy_stride = token_rows(torch.zeros(shape, device=dev, dtype=s.dtype) if dy is None else dy.to(s.dtype))
        dsr, ds_stride = (None, 0) if ds is None else token_rows(ds.to(s.dtype))
        dx = torch.empty(shape, device=dev, dtype=s.dtype) if need_x or need_r else None
        dw = torch.empty(n, device=dev, dtype=w_dtype) if need_w else None
        db = torch.empty(n, device=dev, dtype=b_dtype) if need_b else None
        lib = _lib.load()
        nbytes = lib.fst_layer_norm_backward_workspace_bytes(dtype, b, length, n) if need_w or need_b else 0
        ws = torch.empty(max(nbytes, 1), device=dev, dtype=torch.uint8)
        P = _lib.ptr
        with torch.cuda.device(dev):
            rc = lib.fst_layer_norm_backward(
                dtype, param_dtype, b, length, n, P(s), s_stride, P(w), P(lens), P(stats), P(dyr), dy_stride,
                P(dsr), ds_stride, P(dx), P(dw), P(db), P(ws), nbytes, _lib.stream_handle(dev))
        _lib.check(rc, "flash_layer_norm backward")
        return dx if need_x else None, dx if need_r else None, dw, db, None, None


def flash_layer_norm(
    x: Tensor,
    weight: Optional[Tensor] = None,
    bias: Optional[Tensor] = None,
    eps: float = 1e-5,
    *,
    residual: Optional[Tensor] = None,
    seqlens: Optional[Tensor] = None,
) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    """Layer norm over the last dimension of `x [.., N]` (bfloat16, float16 or
    float32; N up to 16384): `(x - mean) / sqrt(var + eps) * weight + bias`.

    `weight` and `bias` `[N]` may be omitted; they are of x's dtype or both
    float32 (parameters kept in full precision), and get gradients of theirs.
    With `residual` (x's shape and dtype) the norm is of the sum `s = x +
    residual`, rounded to x's dtype, and `(y, s)` is returned: the block's
    output added to the stream, and the stream normalised for the next one, in
    one pass. With `seqlens` `[B]` x is a padded `[B, L, N]`: rows past an
    event's length are not read, come back as zeros in y, s and every
    gradient, and add nothing to the parameters' gradients. `seqlens` `[1]` also
    goes with packed rows `[T, N]`, of which the first `seqlens[0]` are tokens.

    Under `torch.autocast` x and residual of different types are taken in the
    wider one (a float32 stream and a 16-bit branch: float32), and parameters of
    another 16-bit type in float32.

    Any strides are taken (rows a fixed stride apart in place, others copied).
    Statistics and sums are float32; results are bitwise reproducible.
    """
    if x.is_cuda and all(t is None or type(t) in PLAIN for t in (x, residual, weight, bias, seqlens)):
        host = _lib.host()
        out = None if host is None else host.layer_norm(x, residual, weight, bias, eps, seqlens)
        if out is not None:
            return out
    check_rows(x, residual, weight, bias, seqlens if seqlens is not None and seqlens.is_cuda else None)
    if autocast_dtype() is not None and all(t is None or t.dtype in BLOCK_DTYPES for t in (residual, weight, bias)):
        wide = x.dtype if residual is None else torch.promote_types(x.dtype, residual.dtype)
        x, residual = x.to(wide), None if residual is None else residual.to(wide)
        if any(t is not None and t.dtype not in (wide, torch.float32) for t in (weight, bias)):
            weight, bias = (None if t is None else t.float() for t in (weight, bias))
    n = x.shape[-1]
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"residual must have x's shape and dtype ({tuple(x.shape)}, {x.dtype}), got "
                         f"{tuple(residual.shape)}, {residual.dtype}")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None and t.shape != (n,):
            raise ValueError(f"{name} must be [N={n}], got {tuple(t.shape)}")
        if t is not None and t.dtype not in (x.dtype, torch.float32):
            raise ValueError(f"{name} must be {x.dtype} or float32, got {t.dtype}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(f"weight and bias must share one dtype, got {weight.dtype} and {bias.dtype}")
    if not eps >= 0:
        raise ValueError(f"eps must not be negative, got {eps}")
    return _LayerNorm.apply(x, residual, weight, bias, float(eps), seqlens)
