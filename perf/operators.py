"""The operators of a transformer block beside its attention, as measurable cases.

Two operators, each forward alone (`"mode": "fwd"`: inference, validation) or
forward and backward (`"mode": "step"`: training):

* `norm`: layer norm of every token, with the residual sum before it where
  `residual` is set (`flash_layer_norm`):
      s = x + r (rounded to its type: the stream the model carries on),
      y = (s - mean(s)) / sqrt(var(s) + eps) * w + b;
* `ffn`: the gated feed-forward block (`flash_gated_feed_forward`):
      y = (act(x Wg^T + bg) * (x Wu^T + bu)) Wd^T + bd.

A case is a dict of plain values:

    op, mode, dtype ("bf16" / "f16" / "f32": x, and the feed-forward's weights),
    batch, length (tokens of an event, padded), lens: "packed" (every row is a
    token: x is [batch * length, dim]), or how the events' lengths are spread
    over a padded [batch, length, dim]: "full" (no lengths given), "uniform"
    (evenly over min(16, length) .. length; rows past them are padding: their
    outputs and gradients are zero, and they add nothing to the weights'),
    dim, hidden and act ("silu", "gelu", "gelu_tanh") and biases (ffn only),
    residual and params (norm only: the type of w and b).

The multiset of lengths belongs to the case, so its work does not depend on
the seed; the seed draws every value and the order of the events.
"""

from __future__ import annotations

import math
from typing import Dict, List, Optional

import torch

own = False

EPS = 1e-5
_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _norm(name, mode, dtype, batch, length, lens, dim, residual=True, params="f32"):
    case = {"op": "norm", "mode": mode, "dtype": dtype, "batch": batch, "length": length, "lens": lens, "dim": dim,
            "residual": residual, "params": params}
    if name:
        case["name"] = name
    return case


def _ffn(name, mode, dtype, batch, length, lens, dim, hidden, act="silu", biases=False):
    case = {"op": "ffn", "mode": mode, "dtype": dtype, "batch": batch, "length": length, "lens": lens, "dim": dim,
            "hidden": hidden, "act": act, "biases": biases}
    if name:
        case["name"] = name
    return case


def listed() -> List[Dict]:
    return [
        # One event between two layers of an event-by-event reconstruction:
        # the smallest call, all latency.
        _norm("norm_event_fwd", "fwd", "bf16", 1, 187, "packed", 384),
        # The headline training batch (256 events of up to 768 pulses, 12 heads
        # of 32): the norm of every sub-layer, with its residual sum.
        _norm("norm_padded_step", "step", "bf16", 256, 768, "uniform", 384),
        # The same stream in float32, packed, at the width of 8 heads of 64.
        _norm("norm_packed_step_f32", "step", "f32", 1, 60001, "packed", 512, residual=False),
        # A width that is neither a power of two nor even, in half precision
        # with parameters of its own type.
        _norm("norm_odd_step_f16", "step", "f16", 16, 500, "full", 1367, residual=False, params="f16"),
        # A summary token per event through a trained block, a few at a time.
        _ffn("ffn_token_fwd", "fwd", "bf16", 1, 4, "packed", 768, 2048, "gelu", True),
        # One event through a trained block.
        _ffn("ffn_event_fwd", "fwd", "bf16", 1, 187, "packed", 384, 1024),
        # A fine-tuning step on a handful of short events, in half precision.
        _ffn("ffn_small_step_f16", "step", "f16", 16, 64, "uniform", 384, 1024, "gelu_tanh", True),
        # The headline batch's forward (validation).
        _ffn("ffn_padded_fwd", "fwd", "bf16", 256, 768, "uniform", 384, 1024, "gelu", True),
        # The headline training step.
        _ffn("ffn_padded_step", "step", "bf16", 256, 768, "uniform", 384, 1024, "silu", True),
        # A step on few long packed events at the width of 16 heads of 48.
        _ffn("ffn_packed_step", "step", "bf16", 5, 1528, "packed", 768, 2048),
        # A step on a large packed batch of a wide model.
        _ffn("ffn_wide_step", "step", "bf16", 1, 65536, "packed", 1024, 2752),
        # The wide-head configuration (8 heads of 64) in float32.
        _ffn("ffn_step_f32", "step", "f32", 4, 4096, "full", 512, 1408),
    ]


def _logint(rng, lo, hi) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case) -> float:
    """Seconds of a pass at rough rates, to hold drawn cases to the listed ones."""
    w = work(case)
    return w["bytes"] / 4e12 + w["flops"] / (1e14 if case["dtype"] == "f32" else 6e14)


def draw(rng) -> Dict:
    op = rng.choice(["norm", "ffn", "ffn"])
    top = max(_cost(c) for c in listed() if c["op"] == op)
    while True:
        mode = rng.choice(["fwd", "step", "step"])
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        batch = _logint(rng, 1, 512)
        length = _logint(rng, 1, 4096)
        lens = rng.choice(["packed", "uniform", "uniform", "full"])
        if batch * length > 250_000:
            continue
        if op == "norm":
            case = _norm("", mode, dtype, batch, length, lens, _logint(rng, 8, 8192), rng.random() < 0.5,
                         rng.choice(["f32", dtype]))
        else:
            case = _ffn("", mode, dtype, batch, length, lens, 8 * _logint(rng, 4, 160), 8 * _logint(rng, 8, 512),
                        rng.choice(["silu", "gelu", "gelu_tanh"]), rng.random() < 0.5)
        if _cost(case) <= top:
            return case


def _lengths(case) -> Optional[List[int]]:
    """The events' lengths (the order is drawn with the inputs), or None where every row is a token."""
    b, top = case["batch"], case["length"]
    if case["lens"] != "uniform":
        return None
    lo = min(16, top)
    return [lo + int((top + 1 - lo) * (i + 0.5) / b) for i in range(b)]


def _inputs(case, seed: int) -> Dict[str, torch.Tensor]:
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    dt, dim = _TYPES[case["dtype"]], case["dim"]
    lead = (case["batch"] * case["length"],) if case["lens"] == "packed" else (case["batch"], case["length"])

    def rn(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    x: Dict[str, torch.Tensor] = {}
    if case["op"] == "norm":
        pt = _TYPES[case["params"]]
        # A residual stream: channels with offsets and scales of their own.
        x["x"] = (rn(*lead, dim) * (0.5 + rn(dim).abs()) + 0.5 * rn(dim)).to(dt)
        if case["residual"]:
            x["r"] = (2.0 * rn(*lead, dim) + rn(dim)).to(dt)
        x["w"] = (1.0 + 0.2 * rn(dim)).to(pt)
        x["b"] = (0.1 * rn(dim)).to(pt)
        if case["mode"] == "step":
            x["dy"] = (0.01 * rn(*lead, dim)).to(dt)
            if case["residual"]:
                x["ds"] = (0.01 * rn(*lead, dim)).to(dt)
    else:
        hidden = case["hidden"]
        # What a norm hands the block, and weights at the usual scale.
        x["x"] = rn(*lead, dim).to(dt)
        x["wg"] = (rn(hidden, dim) / dim ** 0.5).to(dt)
        x["wu"] = (rn(hidden, dim) / dim ** 0.5).to(dt)
        x["wd"] = (rn(dim, hidden) / hidden ** 0.5).to(dt)
        if case["biases"]:
            x["bg"] = (0.1 * rn(hidden)).to(dt)
            x["bu"] = (0.1 * rn(hidden)).to(dt)
            x["bd"] = (0.1 * rn(dim)).to(dt)
        if case["mode"] == "step":
            x["dy"] = (0.05 * rn(*lead, dim)).to(dt)
    lens = _lengths(case)
    if lens is not None:
        order = torch.randperm(len(lens), generator=host)
        x["lens"] = torch.tensor(lens, dtype=torch.int32)[order].to(dev)
    return x


_LEAVES = {"norm": ("x", "r", "w", "b"), "ffn": ("x", "wg", "wu", "wd", "bg", "bu", "bd")}


def prepare(case, seed: int) -> Dict:
    x = _inputs(case, seed)
    if own and case["mode"] == "step":
        for name in _LEAVES[case["op"]]:
            if name in x:
                x[name].requires_grad_(True)
    return {"case": case, "x": x}


def run(state):
    """One forward, or one forward and backward: the outputs, then the
    gradients of x (and the residual), the weights and the biases."""
    case, x = state["case"], state["x"]
    if own:
        return _own(case, x)
    return _plain_norm(case, x) if case["op"] == "norm" else _plain_ffn(case, x)


def _own(case, x):
    from flash_spacetime_amd import flash_gated_feed_forward, flash_layer_norm

    step = case["mode"] == "step"
    if case["op"] == "norm":
        out = flash_layer_norm(x["x"], x["w"], x["b"], EPS, residual=x.get("r"), seqlens=x.get("lens"))
    else:
        out = flash_gated_feed_forward(x["x"], x["wg"], x["wu"], x["wd"], x.get("bg"), x.get("bu"), x.get("bd"),
                                       case["act"], seqlens=x.get("lens"))
    outs = list(out) if isinstance(out, tuple) else [out]
    if not step:
        return outs
    leaves = [x[n] for n in _LEAVES[case["op"]] if n in x]
    grads = torch.autograd.grad(outs, leaves, [x["dy"], x["ds"]] if "ds" in x else [x["dy"]])
    return [o.detach() for o in outs] + list(grads)


def _padding(case, x, like) -> Optional[torch.Tensor]:
    """[batch, length, 1], true past the events' lengths; None without lengths."""
    if "lens" not in x:
        return None
    return (torch.arange(case["length"], device=like.device)[None, :] >= x["lens"][:, None])[..., None]


def _plain_norm(case, x):
    dt, pt = x["x"].dtype, x["w"].dtype
    pad = _padding(case, x, x["x"])

    def rows(t):
        t = t.float()
        return t if pad is None else t.masked_fill(pad, 0.0)

    s = rows(x["x"])
    if case["residual"]:
        s = (s + rows(x["r"])).to(dt).float()
    w, b = x["w"].float(), x["b"].float()
    c = s - s.mean(-1, keepdim=True)
    rstd = (c.square().mean(-1, keepdim=True) + EPS).rsqrt()
    xhat = c * rstd
    y = rows(xhat * w + b)
    outs = [y.to(dt)] + ([s.to(dt)] if case["residual"] else [])
    if case["mode"] == "fwd":
        return outs
    dy = rows(x["dy"])
    g = dy * w
    dx = rstd * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
    if case["residual"]:
        dx = dx + rows(x["ds"])
    lead = tuple(range(dx.dim() - 1))
    dx = dx.to(dt)
    outs += [dx, dx.clone()] if case["residual"] else [dx]
    return outs + [(dy * xhat).sum(lead).to(pt), dy.sum(lead).to(pt)]


def _plain_ffn(case, x):
    dt = x["x"].dtype
    pad = _padding(case, x, x["x"])

    def rows(t):
        t = t.float()
        return (t if pad is None else t.masked_fill(pad, 0.0)).reshape(-1, t.shape[-1])

    xs, wg, wu, wd = rows(x["x"]), x["wg"].float(), x["wu"].float(), x["wd"].float()
    a, u = xs @ wg.t(), xs @ wu.t()
    if case["biases"]:
        a, u = a + x["bg"].float(), u + x["bu"].float()
    if case["act"] == "silu":
        gate = torch.sigmoid(a)
        act = a * gate
    elif case["act"] == "gelu":
        gate = 0.5 * (1.0 + torch.erf(a * 0.5 ** 0.5))
        act = a * gate
    else:
        t = torch.tanh((2.0 / math.pi) ** 0.5 * (a + 0.044715 * a * a * a))
        act = 0.5 * a * (1.0 + t)
    h = act * u
    y = h @ wd.t()
    if case["biases"]:
        y = y + x["bd"].float()
    y = y.reshape(x["x"].shape)
    if pad is not None:
        y = y.masked_fill(pad, 0.0)
    outs = [y.to(dt)]
    if case["mode"] == "fwd":
        return outs
    dy = rows(x["dy"])
    dh = dy @ wd
    if case["act"] == "silu":
        slope = gate * (1.0 + a * (1.0 - gate))
    elif case["act"] == "gelu":
        slope = gate + a * torch.exp(-0.5 * a * a) * (2.0 * math.pi) ** -0.5
    else:
        slope = 0.5 * (1.0 + t) + 0.5 * a * (1.0 - t * t) * (2.0 / math.pi) ** 0.5 * (1.0 + 3 * 0.044715 * a * a)
    da, du = dh * u * slope, dh * act
    dx = (da @ wg + du @ wu).reshape(x["x"].shape)
    outs += [dx.to(dt), (da.t() @ xs).to(dt), (du.t() @ xs).to(dt), (dy.t() @ h).to(dt)]
    if case["biases"]:
        outs += [da.sum(0).to(dt), du.sum(0).to(dt), dy.sum(0).to(dt)]
    return outs


def work(case) -> Dict[str, float]:
    """Each valid row read once, every row of the outputs written once (padding
    rows are zeros the operator writes), and the definition's operations over
    the valid rows."""
    lens = _lengths(case)
    rows = case["batch"] * case["length"]
    valid = rows if lens is None else sum(lens)
    es = 4 if case["dtype"] == "f32" else 2
    dim, step = case["dim"], case["mode"] == "step"
    if case["op"] == "norm":
        wide = 2 if case["residual"] else 1
        ps = 4 if case["params"] == "f32" else 2
        nbytes = wide * dim * es * (valid + rows) + 2 * dim * ps
        flops = (8 if case["residual"] else 7) * valid * dim
        if step:
            # dy and ds in; one dx (the residual's gradient is the same), dw and db out.
            nbytes += dim * es * (wide * valid + rows) + 2 * dim * ps
            flops += 14 * valid * dim
        return {"bytes": float(nbytes), "flops": float(flops)}
    hidden = case["hidden"]
    weights = 3 * dim * hidden + ((2 * hidden + dim) if case["biases"] else 0)
    nbytes = es * (dim * (valid + rows) + weights)
    flops = 6.0 * valid * dim * hidden
    if step:
        nbytes += es * (dim * (valid + rows) + weights)
        flops += 12.0 * valid * dim * hidden
    return {"bytes": float(nbytes), "flops": flops}


# ---------------------------------------------------------------------------
# The same results in 64 bits, from the definitions: the valid rows gathered,
# the gradients by differentiating the definition, the rows put back.
# ---------------------------------------------------------------------------


def exact(case, seed: int) -> Optional[List[torch.Tensor]]:
    x = _inputs(case, seed)
    step = case["mode"] == "step"
    shape = x["x"].shape
    valid = torch.ones(shape[:-1], dtype=torch.bool, device=x["x"].device)
    if "lens" in x:
        for i, n in enumerate(x["lens"].tolist()):
            valid[i, n:] = False

    def back(t):
        full = torch.zeros(shape, dtype=torch.float64, device=t.device)
        full[valid] = t.detach()
        return full

    def leaf(name, t=None):
        t = x[name] if t is None else t
        return t.double().requires_grad_(step)

    if case["op"] == "norm":
        s = x["x"][valid]
        if case["residual"]:
            s = (s.float() + x["r"][valid].float()).to(s.dtype)
        s, w, b = leaf("x", s), leaf("w"), leaf("b")
        dev = s - s.sum(-1, keepdim=True) / case["dim"]
        y = dev / torch.sqrt((dev * dev).sum(-1, keepdim=True) / case["dim"] + EPS) * w + b
        outs = [back(y)] + ([back(s)] if case["residual"] else [])
        if not step:
            return outs
        ds, dw, db = torch.autograd.grad(y, (s, w, b), x["dy"][valid].double())
        if case["residual"]:
            ds = ds + x["ds"][valid].double()
        ds = back(ds)
        return outs + ([ds, ds.clone()] if case["residual"] else [ds]) + [dw, db]

    leaves = {n: leaf(n) for n in _LEAVES["ffn"][1:] if n in x}
    tokens = leaf("x", x["x"][valid])
    gate = torch.addmm(leaves["bg"], tokens, leaves["wg"].t()) if case["biases"] else tokens @ leaves["wg"].t()
    up = torch.addmm(leaves["bu"], tokens, leaves["wu"].t()) if case["biases"] else tokens @ leaves["wu"].t()
    if case["act"] == "silu":
        gate = gate / (1.0 + torch.exp(-gate))
    elif case["act"] == "gelu":
        gate = gate * torch.erfc(-gate / math.sqrt(2.0)) / 2.0
    else:
        # gelu_tanh: x sigmoid(2 z) = x (1 + tanh z) / 2
        gate = gate / (1.0 + torch.exp(-2.0 * math.sqrt(2.0 / math.pi) * (gate + 0.044715 * gate ** 3)))
    y = (gate * up) @ leaves["wd"].t()
    if case["biases"]:
        y = y + leaves["bd"]
    outs = [back(y)]
    if not step:
        return outs
    grads = torch.autograd.grad(y, (tokens, *leaves.values()), x["dy"][valid].double())
    return outs + [back(grads[0])] + list(grads[1:])
