"""The transformer-block operators' definitions in 64 bits, for the parity tests."""

from __future__ import annotations

import math

import torch

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def valid_rows(shape, seqlens):
    """Bool `shape[:-1]`: rows within their event's length (all without lengths)."""
    if seqlens is None:
        return torch.ones(shape[:-1], dtype=torch.bool)
    lens = torch.as_tensor(seqlens).clamp(0, shape[1])
    return torch.arange(shape[1])[None, :] < lens[:, None]


def norm64(x, residual, weight, bias, eps, valid, dy=None, ds=None):
    """(y, s, dx, dw, db) in float64 on the CPU; rows not valid are zeros. x,
    residual, dy, ds in the operator's type (s is rounded to it)."""
    s = x.cpu()
    if residual is not None:
        s = (s.float() + residual.cpu().float()).to(s.dtype)
    s = torch.where(valid[..., None], s, torch.zeros_like(s)).double()
    n = s.shape[-1]
    w = torch.ones(n, dtype=torch.float64) if weight is None else weight.detach().cpu().double()
    b = torch.zeros(n, dtype=torch.float64) if bias is None else bias.detach().cpu().double()
    c = s - s.mean(-1, keepdim=True)
    rstd = (c.square().mean(-1, keepdim=True) + eps).rsqrt()
    xhat = c * rstd
    y = torch.where(valid[..., None], xhat * w + b, 0.0)
    if dy is None:
        return y, s
    g = torch.where(valid[..., None], dy.detach().cpu().double(), 0.0)
    gw = g * w
    dx = rstd * (gw - gw.mean(-1, keepdim=True) - xhat * (gw * xhat).mean(-1, keepdim=True))
    if ds is not None:
        dx = dx + torch.where(valid[..., None], ds.detach().cpu().double(), 0.0)
    lead = tuple(range(dx.dim() - 1))
    return y, s, dx, (g * xhat).sum(lead), g.sum(lead)


def act64(kind, a):
    """The activation and its derivative."""
    if kind == "silu":
        s = torch.sigmoid(a)
        return a * s, s * (1 + a * (1 - s))
    if kind == "gelu":
        phi = 0.5 * torch.erfc(-a / math.sqrt(2))
        return a * phi, phi + a * torch.exp(-a * a / 2) / math.sqrt(2 * math.pi)
    z = math.sqrt(2 / math.pi) * (a + 0.044715 * a ** 3)
    s = torch.sigmoid(2 * z)
    return a * s, s + a * s * (1 - s) * 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * a * a)


def ffn64(x, wg, wu, wd, bg, bu, bd, kind, valid, dy=None):
    """(y,) or (y, dx, dwg, dwu, dwd, dbg, dbu, dbd) in float64 on x's device; rows
    not valid are zeros."""
    dev = x.device
    valid = valid.to(dev)
    d = lambda t: 0.0 if t is None else t.detach().double()  # noqa: E731
    xs = x.detach()[valid].double()
    a, u = xs @ d(wg).t() + d(bg), xs @ d(wu).t() + d(bu)
    act, slope = act64(kind, a)
    h = act * u

    def back(rows):
        full = torch.zeros(x.shape, dtype=torch.float64, device=dev)
        full[valid] = rows
        return full

    y = back(h @ d(wd).t() + d(bd))
    if dy is None:
        return (y,)
    g = dy.detach()[valid].double()
    dh = g @ d(wd)
    da, du = dh * u * slope, dh * act
    return (y, back(da @ d(wg) + du @ d(wu)), da.t() @ xs, du.t() @ xs, g.t() @ h, da.sum(0), du.sum(0), g.sum(0))
