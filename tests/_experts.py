"""The RMS norm's and the mixture of experts' definitions in 64 bits, for the parity tests."""

from __future__ import annotations

import torch

from tests._block import act64


def rms64(x, residual, weight, eps, valid, dy=None, ds=None):
    """(y, s, rstd) or (y, s, rstd, dx, dw) in float64 on the CPU; rows not valid are
    zeros. x, residual, dy, ds in the operator's type (s is rounded to it)."""
    s = x.detach().cpu()
    if residual is not None:
        s = (s.float() + residual.detach().cpu().float()).to(s.dtype)
    s = torch.where(valid[..., None], s, torch.zeros_like(s)).double()
    w = torch.ones(s.shape[-1], dtype=torch.float64) if weight is None else weight.detach().cpu().double()
    rstd = (s.square().mean(-1, keepdim=True) + eps).rsqrt()
    xhat = torch.where(valid[..., None], s * rstd, 0.0)
    if dy is None:
        return xhat * w, s, rstd
    g = torch.where(valid[..., None], dy.detach().cpu().double(), 0.0)
    gw = g * w
    dx = rstd * (gw - xhat * (gw * xhat).mean(-1, keepdim=True))
    dx = torch.where(valid[..., None], dx, 0.0)
    if ds is not None:
        dx = dx + torch.where(valid[..., None], ds.detach().cpu().double(), 0.0)
    return xhat * w, s, rstd, dx, (g * xhat).sum(tuple(range(dx.dim() - 1)))


def route64(logits, top_k, normalize, valid, dw=None):
    """(weights, experts) or (weights, experts, dlogits): rows not valid have expert -1."""
    v = logits.detach().cpu().double()
    key = torch.where(v.isnan(), float("inf"), v)
    # NaN ranks above +inf; of equal ones the lowest index first
    at = torch.sort(-key, dim=-1, stable=True).indices
    at = torch.gather(at, -1, torch.sort((~torch.gather(v.isnan(), -1, at)).int(), dim=-1, stable=True).indices)[..., :top_k]
    best = torch.gather(v, -1, at)
    none = (best == -torch.inf) | ~valid[..., None]
    top = torch.where(none[..., :1], 0.0, best[..., :1])
    e = torch.where(none, 0.0, torch.exp(best - top))
    total = torch.where(v == -torch.inf, 0.0, torch.exp(v - top)).sum(-1, keepdim=True) if not normalize else e.sum(-1, keepdim=True)
    weights = torch.where(none, 0.0, e / total)
    experts = torch.where(none, -1, at)
    if dw is None:
        return weights, experts
    g = torch.where(none, 0.0, dw.detach().cpu().double())
    mean = (weights * g).sum(-1, keepdim=True)
    grad = torch.zeros_like(v).scatter_add(-1, at, torch.where(none, 0.0, weights * (g - mean if normalize else g)))
    if not normalize:
        p = torch.where((v == -torch.inf) | none[..., :1], 0.0, torch.exp(v - top) / total)
        grad = grad - mean * p
    return weights, experts, grad


def sorted64(experts, n):
    """(order, place, offsets) by a stable sort on the CPU."""
    flat = experts.detach().cpu().long().reshape(-1)
    ids = torch.where((flat < 0) | (flat >= n), n, flat)
    ids, order = torch.sort(ids, stable=True)
    rows = torch.arange(ids.numel())
    place = torch.empty_like(rows)
    place[order] = torch.where(ids == n, -1, rows)
    offsets = torch.tensor([int((ids < e).sum()) for e in range(n + 1)])
    return torch.where(ids == n, -1, order).int(), place.reshape(experts.shape).int(), offsets.int()


def expert_ffn64(x, offsets, wg, wu, wd, kind, dy=None):
    """(y,) or (y, dx, dwg, dwu, dwd) in float64 on x's device."""
    y = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    dx, grads = torch.zeros_like(y), [torch.zeros(w.shape, dtype=torch.float64, device=x.device) for w in (wg, wu, wd)]
    ends = offsets.tolist()
    for e, (lo, hi) in enumerate(zip(ends, ends[1:])):
        if lo == hi:
            continue
        xs, g, u, d = x[lo:hi].detach().double(), *(w[e].detach().double() for w in (wg, wu, wd))
        a, b = xs @ g.t(), xs @ u.t()
        act, slope = act64(kind, a)
        h = act * b
        y[lo:hi] = h @ d.t()
        if dy is not None:
            t = dy[lo:hi].detach().double()
            dh = t @ d
            da, du = dh * b * slope, dh * act
            dx[lo:hi] = da @ g + du @ u
            for full, v in zip(grads, (da.t() @ xs, du.t() @ xs, t.t() @ h)):
                full[e] = v
    return (y,) if dy is None else (y, dx, *grads)
