"""Gated feed-forward block of token rows, for packed rows and padded batches.

The other half of a transformer block beside its attention (graphnet's
`Block_rel` around the reference's operator, reference README.md:105-116), with a
gate: both projections, the activation and their product in one kernel, the
output projection in another, and the backward on the same matrix-core kernels
(`fst_ffn_forward`, `fst_ffn_backward`). No reference counterpart.
"""

from __future__ import annotations

from typing import Any, Optional

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _lib
from .norm import BLOCK_DTYPES, PLAIN, autocast_dtype, batch_of_rows, check_rows, token_rows

ACTIVATIONS = {"silu": _lib.FST_SILU, "gelu": _lib.FST_GELU, "gelu_tanh": _lib.FST_GELU_TANH}


def _dense(t: Optional[Tensor]) -> Optional[Tensor]:
    """A weight or bias as the kernels read it: contiguous, on a multiple of 16 bytes."""
    if t is None:
        return None
    t = t.contiguous()
    return t.clone() if t.data_ptr() % 16 else t


class _GatedFeedForward(torch.autograd.Function):
    """Fused forward and deterministic backward; keeps x, the hidden rows and, in
    float32, both projections (16-bit types form them again, unrounded)."""

    @staticmethod
    def forward(ctx: Any, x, w_gate, w_up, w_down, b_gate, b_up, b_down, activation, seqlens):  # type: ignore[override]
        dtype, act = BLOCK_DTYPES[x.dtype], ACTIVATIONS[activation]
        b, length, lens = batch_of_rows(x, seqlens)
        f, d = w_gate.shape
        xr, x_stride = token_rows(x, 16)
        wg, wu, wd, bg, bu, bd = (_dense(t) for t in (w_gate, w_up, w_down, b_gate, b_up, b_down))
        keep = any(ctx.needs_input_grad)
        like = {"device": x.device, "dtype": x.dtype}
        y = torch.empty(x.shape, **like)
        hidden = torch.empty(b * length, f, **like)
        gate, up = (torch.empty_like(hidden), torch.empty_like(hidden)) if keep and dtype == _lib.FST_F32 else (None, None)
        rowmap = None if lens is None else torch.empty(b * length + 1, device=x.device, dtype=torch.int32)
        P = _lib.ptr
        with torch.cuda.device(x.device):
            rc = _lib.load().fst_ffn_forward(
                dtype, act, b, length, d, f, P(xr), x_stride, P(wg), P(wu), P(wd), P(bg), P(bu), P(bd), P(lens),
                P(hidden), P(gate), P(up), P(rowmap), P(y), _lib.stream_handle(x.device))
        _lib.check(rc, "flash_gated_feed_forward")
        if keep:
            ctx.save_for_backward(xr, wg, wu, wd, bg, bu, lens, hidden, gate, up, rowmap)
            ctx.meta = (dtype, act, b, length, d, f, x_stride, x.shape)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, dy: Tensor):  # type: ignore[override]
        x, wg, wu, wd, bg, bu, lens, hidden, gate, up, rowmap = ctx.saved_tensors
        dtype, act, b, length, d, f, x_stride, shape = ctx.meta
        _lib.refuse_fx_recording()
        need = ctx.needs_input_grad[:7]
        like = {"device": x.device, "dtype": x.dtype}
        dyr, dy_stride = token_rows(dy.to(x.dtype), 16)
        shapes = (shape, (f, d), (f, d), (d, f), (f,), (f,), (d,))
        grads = [torch.empty(s, **like) if n else None for s, n in zip(shapes, need)]
        lib = _lib.load()
        nbytes = lib.fst_ffn_backward_workspace_bytes(dtype, b, length, d, f)
        ws = torch.empty(max(nbytes, 1), device=x.device, dtype=torch.uint8)
        P = _lib.ptr
        with torch.cuda.device(x.device):
            rc = lib.fst_ffn_backward(
                dtype, act, b, length, d, f, P(x), x_stride, P(wg), P(wu), P(wd), P(bg), P(bu), P(lens), P(hidden),
                P(gate), P(up), P(rowmap), P(dyr), dy_stride, *(P(g) for g in grads), P(ws), nbytes, _lib.stream_handle(x.device))
        _lib.check(rc, "flash_gated_feed_forward backward")
        return (*grads, None, None)


def flash_gated_feed_forward(
    x: Tensor,
    w_gate: Tensor,
    w_up: Tensor,
    w_down: Tensor,
    b_gate: Optional[Tensor] = None,
    b_up: Optional[Tensor] = None,
    b_down: Optional[Tensor] = None,
    activation: str = "silu",
    *,
    seqlens: Optional[Tensor] = None,
) -> Tensor:
    """`(act(x w_gate^T + b_gate) * (x w_up^T + b_up)) w_down^T + b_down`.

    `x` is `[.., D]` in bfloat16, float16 or float32; `w_gate`, `w_up` `[F, D]` and
    `w_down` `[D, F]` (nn.Linear layout) and the biases (each may be omitted)
    share its dtype. D and F are multiples of 8. `activation` is "silu", "gelu"
    (with the normal distribution function) or "gelu_tanh". With `seqlens` `[B]` x
    is a padded `[B, L, D]`: rows past an event's length are neither read nor
    computed, come back as zeros in the output and x's gradient, and add
    nothing to the weights' gradients (`seqlens` `[1]` also goes with packed rows `[T,
    D]`, of which the first `seqlens[0]` are tokens).

    Under `torch.autocast` tensors of different types are taken in autocast's
    (16-bit rows beside float32 weights); of one type they stay in it.

    Products accumulate in float32 on the matrix cores. bfloat16 and float16
    round the hidden rows to their type between the products (float16 ones past
    65504 are infinite) and the projections' gradients in the backward, which
    forms the projections again, unrounded; float32 keeps them. "gelu" takes the
    distribution function to 1e-7. Results are bitwise reproducible.

    Memory is for all rows of x, padding among them: the call keeps F elements a row
    for the backward (float32 3 F), which takes another 2 F.
    """
    tensors = (x, w_gate, w_up, w_down, b_gate, b_up, b_down)
    if x.is_cuda and activation in ACTIVATIONS and all(t is None or type(t) in PLAIN for t in (*tensors, seqlens)):
        host = _lib.host()
        out = None if host is None else host.feed_forward(*tensors, ACTIVATIONS[activation], seqlens)
        if out is not None:
            return out
    check_rows(x, w_gate, w_up, w_down, b_gate, b_up, b_down,
               seqlens if seqlens is not None and seqlens.is_cuda else None)
    low, types = autocast_dtype(), {t.dtype for t in tensors if t is not None}
    if low is not None and len(types) > 1 and types <= BLOCK_DTYPES.keys():
        tensors = tuple(None if t is None else t.to(low) for t in tensors)
        return flash_gated_feed_forward(*tensors, activation, seqlens=seqlens)
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    d = x.shape[-1]
    if w_gate.dim() != 2 or w_gate.shape[1] != d:
        raise ValueError(f"w_gate must be [F, D={d}], got {tuple(w_gate.shape)}")
    f = w_gate.shape[0]
    for name, t, shape in (("w_up", w_up, (f, d)), ("w_down", w_down, (d, f)), ("b_gate", b_gate, (f,)),
                           ("b_up", b_up, (f,)), ("b_down", b_down, (d,))):
        if t is not None and t.shape != shape:
            raise ValueError(f"{name} must be {list(shape)}, got {tuple(t.shape)}")
    for name, t in (("w_gate", w_gate), ("w_up", w_up), ("w_down", w_down), ("b_gate", b_gate), ("b_up", b_up),
                    ("b_down", b_down)):
        if t is not None and t.dtype != x.dtype:
            raise ValueError(f"{name} must have x's dtype {x.dtype}, got {t.dtype}")
    return _GatedFeedForward.apply(x, w_gate, w_up, w_down, b_gate, b_up, b_down, activation, seqlens)
