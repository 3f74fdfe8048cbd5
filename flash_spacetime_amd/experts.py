"""Mixture of experts in the feed-forward's place, for packed rows and padded batches.

The steps of it, each an operator: a router's choice of experts for every token
(`flash_expert_route`), the tokens' slots sorted by expert (`flash_expert_sort`),
their rows brought into that order and the experts' rows back to the tokens
(`flash_expert_dispatch`, `flash_expert_combine`), and between them the gated
feed-forward of each expert on its rows (`flash_expert_feed_forward`, the kernels of
`feed_forward.py` over runs of rows). HIP kernels behind the C ABI
(`fst_expert_*`). Counts of rows stay on the device: nothing waits for the GPU, and a
batch of the same shape can be replayed from a graph. No reference counterpart.
"""

from __future__ import annotations

from typing import Any, NamedTuple, Optional, Tuple

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _lib
from .feed_forward import ACTIVATIONS, _dense
from .norm import BLOCK_DTYPES, PLAIN, autocast_dtype, batch_of_rows, check_rows, token_rows


class ExpertOrder(NamedTuple):
    """The tokens' slots sorted by expert (int32 tensors): `order [slots]`, the slot of
    each sorted row, -1 past the last expert's; `place [.., K]`, the row of each token's
    slots, -1 where they have no expert; `offsets [experts + 1]`, the first row of each
    expert and behind the last.

    `flash_expert_dispatch` and `flash_expert_combine` take a slot to have a row where its
    place lies below `offsets[-1]`. Slots may be taken out after the sort (place -1, experts
    cut off the end of `offsets`): they then read and write nothing, and the rows that they
    had are zeros wherever rows are written. Otherwise order and place belong to each other,
    `place[order[r]] = r`: no two slots share a row."""

    order: Tensor
    place: Tensor
    offsets: Tensor


# --- router -----------------------------------------------------------------


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, logits, top_k, normalize, seqlens):  # type: ignore[override]
        dtype = BLOCK_DTYPES[logits.dtype]
        b, length, lens = batch_of_rows(logits, seqlens)
        rows, stride = token_rows(logits)
        shape = (*logits.shape[:-1], top_k)
        weights = torch.empty(shape, device=logits.device, dtype=torch.float32)
        experts = torch.empty(shape, device=logits.device, dtype=torch.int32)
        P = _lib.ptr
        with torch.cuda.device(logits.device):
            rc = _lib.load().fst_expert_route(dtype, b, length, logits.shape[-1], top_k, normalize, P(rows), stride, P(lens),
                                              P(weights), P(experts), _lib.stream_handle(logits.device))
        _lib.check(rc, "flash_expert_route")
        ctx.mark_non_differentiable(experts)
        ctx.set_materialize_grads(False)
        if ctx.needs_input_grad[0]:
            ctx.save_for_backward(None if normalize else rows, lens, weights, experts)
            ctx.meta = (dtype, b, length, logits.shape, top_k, normalize, stride, logits.dtype)
        return weights, experts

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, dw: Optional[Tensor], _=None):  # type: ignore[override]
        if dw is None:
            return (None,) * 4
        _lib.refuse_fx_recording()
        rows, lens, weights, experts = ctx.saved_tensors
        dtype, b, length, shape, top_k, normalize, stride, kind = ctx.meta
        dw = dw.float().contiguous()
        dlogits = torch.empty(shape, device=dw.device, dtype=kind)
        P = _lib.ptr
        with torch.cuda.device(dw.device):
            rc = _lib.load().fst_expert_route_backward(
                dtype, b, length, shape[-1], top_k, normalize, P(rows), stride, P(lens), P(weights), P(experts), P(dw),
                P(dlogits), _lib.stream_handle(dw.device))
        _lib.check(rc, "flash_expert_route backward")
        return dlogits, None, None, None


def flash_expert_route(
    logits: Tensor,
    top_k: int,
    *,
    normalize: bool = True,
    seqlens: Optional[Tensor] = None,
) -> Tuple[Tensor, Tensor]:
    """Each token's `top_k` experts and their weights, from `logits [.., E]`
    (bfloat16, float16 or float32; E up to 512, top_k up to 16).

    Returns `(weights, experts)`, `[.., top_k]` in float32 and int32: the largest
    logits by falling value, of equal ones the lowest index first, and their
    softmax over the chosen experts, or with `normalize=False` over all E. A logit of
    -inf is never chosen: slots that find none are expert -1 with weight 0. NaN ranks
    highest and makes the token's weights NaN. With `seqlens` `[B]` the logits are a
    padded `[B, L, E]` (`[1]`: packed `[T, E]`): rows past an event's length have no
    expert.

    The weights' gradient reaches the logits; float32 inside, bitwise reproducible.
    """
    if logits.is_cuda and all(t is None or type(t) in PLAIN for t in (logits, seqlens)) and type(top_k) is int:
        host = _lib.host()
        out = None if host is None else host.expert_route(logits, top_k, bool(normalize), seqlens)
        if out is not None:
            return out
    check_rows(logits, seqlens if seqlens is not None and seqlens.is_cuda else None)
    if isinstance(top_k, bool) or not isinstance(top_k, int) or not 1 <= top_k <= logits.shape[-1]:
        raise ValueError(f"top_k must be an integer of 1 .. {logits.shape[-1]} experts, got {top_k!r}")
    return _Route.apply(logits, top_k, bool(normalize), seqlens)


# --- sort -------------------------------------------------------------------


class _Sort(torch.autograd.Function):
    """An autograd function for its records: torch's tracer takes it as a call."""

    @staticmethod
    def forward(ctx: Any, experts, num_experts):  # type: ignore[override]
        slots = experts.numel()
        if experts.dtype != torch.int32:
            experts = experts.long().clamp(-1, num_experts).int()
        experts = experts.contiguous()
        like = {"device": experts.device, "dtype": torch.int32}
        order, place = torch.empty(slots, **like), torch.empty(experts.shape, **like)
        offsets = torch.empty(num_experts + 1, **like)
        lib = _lib.load()
        nbytes = lib.fst_expert_sort_workspace_bytes(slots, num_experts)
        ws = torch.empty(max(nbytes, 1), device=experts.device, dtype=torch.uint8)
        P = _lib.ptr
        with torch.cuda.device(experts.device):
            rc = lib.fst_expert_sort(slots, num_experts, P(experts), P(order), P(place), P(offsets), P(ws), nbytes,
                                     _lib.stream_handle(experts.device))
        _lib.check(rc, "flash_expert_sort")
        ctx.mark_non_differentiable(order, place, offsets)
        return order, place, offsets


def flash_expert_sort(experts: Tensor, num_experts: int) -> ExpertOrder:
    """The slots of `experts [.., K]` (integers) sorted by expert, those of one expert in
    the order they stand in. Values outside 0 .. num_experts - 1 are no expert:
    their slots get no row."""
    if experts.is_cuda and type(experts) in PLAIN and type(num_experts) is int:
        host = _lib.host()
        out = None if host is None else host.expert_sort(experts, num_experts)
        if out is not None:
            return ExpertOrder(*out)
    _lib.refuse_fx_recording()
    _lib.require_gpu(experts)
    if experts.dtype.is_floating_point or experts.dtype.is_complex or experts.dtype == torch.bool:
        raise ValueError(f"experts must be an integer tensor, got {experts.dtype}")
    if experts.dim() < 1:
        raise ValueError("experts must be [.., K], got a scalar")
    if isinstance(num_experts, bool) or not isinstance(num_experts, int) or num_experts < 1:
        raise ValueError(f"num_experts must be a positive integer, got {num_experts!r}")
    if experts.numel() > 0x7FFFFFFF:
        raise ValueError(f"too many slots ({experts.numel()})")
    return ExpertOrder(*_Sort.apply(experts, num_experts))


# --- rows to the experts and back -------------------------------------------


def _spread(what, x, place, offsets, weights=None, back=None, rows=None, out=True):
    """(rows at their places, dots with back): fst_expert_spread."""
    n, k = x.shape[-1], place.shape[-1]
    xr, x_stride = token_rows(x)
    br, b_stride = (None, 0) if back is None else token_rows(back)
    rows = place.numel() if rows is None else rows
    o = torch.zeros(rows, n, device=x.device, dtype=x.dtype) if out else None  # rows may be no slot's
    dw = None if back is None else torch.empty(place.shape, device=x.device, dtype=weights.dtype)
    dtype = BLOCK_DTYPES[x.dtype]
    P = _lib.ptr
    with torch.cuda.device(x.device):
        rc = _lib.load().fst_expert_spread(
            dtype, dtype if weights is None else BLOCK_DTYPES[weights.dtype], place.numel() // k, k, n, rows, P(xr), x_stride,
            P(place), offsets.data_ptr() + 4 * (int(offsets.numel()) - 1), P(weights), P(br), b_stride, P(o), P(dw),
            _lib.stream_handle(x.device))
    _lib.check(rc, what)
    return o, dw


def _gather(what, x, place, weights=None):
    """The sums of rows at their places: fst_expert_gather."""
    n, k = x.shape[-1], place.shape[-1]
    xr, x_stride = token_rows(x)
    out = torch.empty(*place.shape[:-1], n, device=x.device, dtype=x.dtype)
    dtype = BLOCK_DTYPES[x.dtype]
    P = _lib.ptr
    with torch.cuda.device(x.device):
        rc = _lib.load().fst_expert_gather(
            dtype, dtype if weights is None else BLOCK_DTYPES[weights.dtype], place.numel() // k, k, n, x.shape[0], P(xr),
            x_stride, P(place), P(weights), P(out), _lib.stream_handle(x.device))
    _lib.check(rc, what)
    return out


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, x, place, offsets):  # type: ignore[override]
        ctx.save_for_backward(place)
        return _spread("flash_expert_dispatch", x, place, offsets)[0]

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, dxs: Tensor):  # type: ignore[override]
        _lib.refuse_fx_recording()
        (place,) = ctx.saved_tensors
        return _gather("flash_expert_dispatch backward", dxs, place), None, None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, ys, weights, place, offsets):  # type: ignore[override]
        w = weights.contiguous()
        ctx.save_for_backward(ys if ctx.needs_input_grad[1] else None, w, place, offsets)
        ctx.meta = ys.shape[0], ys.dtype
        return _gather("flash_expert_combine", ys, place, w)

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, dy: Tensor):  # type: ignore[override]
        _lib.refuse_fx_recording()
        ys, w, place, offsets = ctx.saved_tensors
        rows, kind = ctx.meta
        dys, dw = _spread("flash_expert_combine backward", dy.to(kind), place, offsets, w, ys, rows, ctx.needs_input_grad[0])
        return dys, dw, None, None


def _check_order(order: ExpertOrder, x: Tensor) -> Tuple[Tensor, Tensor]:
    """(place, offsets) of an order on x's device; places from offsets[-1] on are -1."""
    if not isinstance(order, ExpertOrder):
        raise ValueError(f"order must be an ExpertOrder (flash_expert_sort), got {type(order).__name__}")
    for name, t in order._asdict().items():
        if not isinstance(t, Tensor) or t.dtype != torch.int32 or t.device != x.device:
            got = f"{t.dtype} on {t.device}" if isinstance(t, Tensor) else type(t).__name__
            raise ValueError(f"order.{name} must be int32 on {x.device}, got {got}")
    if order.place.dim() < 1 or order.place.shape[-1] < 1 or order.offsets.dim() != 1 or order.offsets.numel() < 2:
        raise ValueError(f"order must have place [.., K] and offsets [experts + 1], got {tuple(order.place.shape)}, "
                         f"{tuple(order.offsets.shape)}")
    place, offsets = order.place.contiguous(), order.offsets.contiguous()
    return place.masked_fill(place >= offsets[-1:], -1), offsets


def flash_expert_dispatch(x: Tensor, order: ExpertOrder) -> Tensor:
    """The tokens' rows `x [.., D]` in the experts' order, `[slots, D]`: row
    `order.place[t, k]` is x's row t. Rows of no slot, those past the last expert's among
    them, are zeros, and a token without experts is not read. x's gradient is the float32 sum over its slots,
    rounded once. Any strides are taken, D up to 16384."""
    if x.is_cuda and type(x) in PLAIN and isinstance(order, ExpertOrder) and isinstance(order.order, Tensor):
        host = _lib.host()
        out = None if host is None else host.expert_dispatch(x, *order)
        if out is not None:
            return out
    check_rows(x)
    place, offsets = _check_order(order, x)
    if x.shape[:-1] != place.shape[:-1]:
        raise ValueError(f"x must be {[*place.shape[:-1], 'D']} as order.place {tuple(place.shape)}, got {tuple(x.shape)}")
    return _Dispatch.apply(x, place, offsets)


def flash_expert_combine(ys: Tensor, weights: Tensor, order: ExpertOrder) -> Tensor:
    """The experts' rows `ys [slots, D]` back at their tokens, weighted and summed:
    `y[t] = sum_k weights[t, k] ys[order.place[t, k]]`, `[.., D]`, summed in float32 and
    rounded once. `weights` is `order.place`'s shape in float32 or ys' dtype; slots without
    an expert add nothing, whatever their weight. ys may be cut behind the last expert's rows,
    or go on behind the slots: a place past its end is none, as it is past `offsets[-1]`. Gradients of ys (zeros in rows of no slot)
    and of the weights."""
    if (ys.is_cuda and type(ys) in PLAIN and type(weights) in PLAIN and isinstance(order, ExpertOrder)
            and isinstance(order.order, Tensor)):
        host = _lib.host()
        out = None if host is None else host.expert_combine(ys, weights, *order)
        if out is not None:
            return out
    check_rows(ys, weights)
    place, offsets = _check_order(order, ys)
    if autocast_dtype() is not None and weights.dtype in BLOCK_DTYPES and weights.dtype != ys.dtype:
        weights = weights.float()
    if ys.dim() != 2:
        raise ValueError(f"ys must be [slots, D], got {tuple(ys.shape)}")
    if weights.shape != place.shape or weights.dtype not in (ys.dtype, torch.float32):
        raise ValueError(f"weights must be {list(place.shape)} in {ys.dtype} or float32, got {tuple(weights.shape)}, "
                         f"{weights.dtype}")
    return _Combine.apply(ys, weights, place, offsets)


# --- the experts' feed-forward ----------------------------------------------


class _ExpertFeedForward(torch.autograd.Function):
    """Fused forward and deterministic backward; keeps x, the hidden rows and, in
    float32, both projections (16-bit types form them again, unrounded)."""

    @staticmethod
    def forward(ctx: Any, x, offsets, w_gate, w_up, w_down, activation):  # type: ignore[override]
        dtype, act = BLOCK_DTYPES[x.dtype], ACTIVATIONS[activation]
        rows = x.shape[0]
        e, f, d = w_gate.shape
        xr, x_stride = token_rows(x, 16)
        wg, wu, wd = (_dense(t) for t in (w_gate, w_up, w_down))
        keep = any(ctx.needs_input_grad)
        like = {"device": x.device, "dtype": x.dtype}
        y = torch.empty(rows, d, **like)
        hidden = torch.empty(rows, f, **like)
        gate, up = (torch.empty_like(hidden), torch.empty_like(hidden)) if keep and dtype == _lib.FST_F32 else (None, None)
        P = _lib.ptr
        with torch.cuda.device(x.device):
            rc = _lib.load().fst_expert_ffn_forward(
                dtype, act, rows, e, d, f, P(xr), x_stride, P(offsets), P(wg), P(wu), P(wd), P(hidden), P(gate), P(up), P(y),
                _lib.stream_handle(x.device))
        _lib.check(rc, "flash_expert_feed_forward")
        if keep:
            ctx.save_for_backward(xr, offsets, wg, wu, wd, hidden, gate, up)
            ctx.meta = (dtype, act, rows, e, d, f, x_stride)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx: Any, dy: Tensor):  # type: ignore[override]
        x, offsets, wg, wu, wd, hidden, gate, up = ctx.saved_tensors
        dtype, act, rows, e, d, f, x_stride = ctx.meta
        _lib.refuse_fx_recording()
        need = [ctx.needs_input_grad[i] for i in (0, 2, 3, 4)]
        like = {"device": x.device, "dtype": x.dtype}
        dyr, dy_stride = token_rows(dy.to(x.dtype), 16)
        shapes = ((rows, d), (e, f, d), (e, f, d), (e, d, f))
        grads = [torch.empty(s, **like) if n else None for s, n in zip(shapes, need)]
        lib = _lib.load()
        nbytes = lib.fst_expert_ffn_backward_workspace_bytes(dtype, rows, e, d, f)
        ws = torch.empty(max(nbytes, 1), device=x.device, dtype=torch.uint8)
        P = _lib.ptr
        with torch.cuda.device(x.device):
            rc = lib.fst_expert_ffn_backward(
                dtype, act, rows, e, d, f, P(x), x_stride, P(offsets), P(wg), P(wu), P(wd), P(hidden), P(gate), P(up), P(dyr),
                dy_stride, *(P(g) for g in grads), P(ws), nbytes, _lib.stream_handle(x.device))
        _lib.check(rc, "flash_expert_feed_forward backward")
        return grads[0], None, *grads[1:], None


def flash_expert_feed_forward(
    x: Tensor,
    offsets: Tensor,
    w_gate: Tensor,
    w_up: Tensor,
    w_down: Tensor,
    activation: str = "silu",
) -> Tensor:
    """`(act(x w_gate[e]^T) * (x w_up[e]^T)) w_down[e]^T` for the rows of each expert e.

    `x` is `[rows, D]` in bfloat16, float16 or float32 with the rows of expert e from
    `offsets[e]` to `offsets[e + 1] - 1` (`offsets [E + 1]` int32, from
    `flash_expert_sort`; E up to 512); `w_gate`, `w_up` `[E, F, D]` and `w_down` `[E, D, F]` share its
    dtype. D and F are multiples of 8. Offsets must not fall; they may be a part of a
    longer table (with its experts' weights). Rows outside these experts' are neither read
    nor computed and come back as zeros in the output and x's gradient; an expert without
    rows gets gradients of zeros. Types, activations, rounding and autocast are
    `flash_gated_feed_forward`'s; there are no biases.

    Memory is for all rows of x: the call keeps F elements a row for the backward (float32
    3 F), which takes another 2 F, and three times the weights.
    """
    tensors = (x, w_gate, w_up, w_down)
    if x.is_cuda and activation in ACTIVATIONS and all(type(t) in PLAIN for t in (*tensors, offsets)):
        host = _lib.host()
        out = None if host is None else host.expert_feed_forward(x, offsets, w_gate, w_up, w_down, ACTIVATIONS[activation])
        if out is not None:
            return out
    check_rows(*tensors, offsets)
    low, types = autocast_dtype(), {t.dtype for t in tensors}
    if low is not None and len(types) > 1 and types <= BLOCK_DTYPES.keys():
        return flash_expert_feed_forward(x.to(low), offsets, *(t.to(low) for t in tensors[1:]), activation)
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    if x.dim() != 2:
        raise ValueError(f"x must be [rows, D], got {tuple(x.shape)}")
    d = x.shape[1]
    if w_gate.dim() != 3 or w_gate.shape[2] != d:
        raise ValueError(f"w_gate must be [E, F, D={d}], got {tuple(w_gate.shape)}")
    e, f = w_gate.shape[:2]
    for name, t, shape in (("w_up", w_up, (e, f, d)), ("w_down", w_down, (e, d, f))):
        if t.shape != shape:
            raise ValueError(f"{name} must be {list(shape)}, got {tuple(t.shape)}")
    for name, t in (("w_gate", w_gate), ("w_up", w_up), ("w_down", w_down)):
        if t.dtype != x.dtype:
            raise ValueError(f"{name} must have x's dtype {x.dtype}, got {t.dtype}")
    if offsets.dtype != torch.int32 or offsets.shape != (e + 1,):
        raise ValueError(f"offsets must be int32 [E + 1 = {e + 1}], got {offsets.dtype} {tuple(offsets.shape)}")
    return _ExpertFeedForward.apply(x, offsets.contiguous(), w_gate, w_up, w_down, activation)
