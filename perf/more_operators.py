"""The block's root-mean-square norm and its mixture of experts, as measurable cases.

Five operators, each forward alone (`"mode": "fwd"`: inference, validation) or
forward and backward (`"mode": "step"`: training):

* `rms`: root-mean-square norm of every token, with the residual sum before it
  where `residual` is set (`flash_rms_norm`):
      s = x + r (rounded to its type: the stream the model carries on),
      y = s / sqrt(mean(s^2) + eps) * w;
* `rms8`: the same norm with its output in 8 bits (e4m3) and one scale a row,
  for the products of a trained model (`flash_rms_norm_fp8`):
      scale = max|y| / 448 (at least 2^-126), q = y / scale;
* `route`: each token's `top` largest logits of `experts` (ties: the lowest
  index), their softmax as weights, and the tokens' slots sorted by expert
  (`flash_expert_route`, `flash_expert_sort`);
* `shuffle`: rows brought into the experts' order, and the experts' rows back
  to their tokens, weighted and summed (`flash_expert_dispatch`,
  `flash_expert_combine`):
      xs[place[t, k]] = x[t],  y[t] = sum_k w[t, k] ys[place[t, k]];
* `experts`: the gated feed-forward of rows in the experts' order
  (`flash_expert_feed_forward`):
      y = (act(x Wg_e^T) * (x Wu_e^T)) Wd_e^T for the rows of expert e.

A case is a dict of plain values:

    op, mode, dtype ("bf16" / "f16" / "f32": rows, logits and the experts'
    weights), batch, length (tokens of an event, padded), lens: "packed" (every
    row is a token: rows are [batch * length, ..]), or how the events' lengths
    are spread over a padded [batch, length, ..]: "full" (no lengths given),
    "uniform" (evenly over min(16, length) .. length; rows past them are
    padding: they go to no expert, and their outputs and gradients are zero),
    dim (but route), residual and params (rms, rms8: the type of w), experts and
    top (route, shuffle, experts), softmax (route: over the "chosen" logits or
    "all"), hidden and act ("silu", "gelu", "gelu_tanh"), and skew (experts: the
    experts' loads lie evenly within 1 - skew .. 1 + skew of their mean, and one of
    more than four gets no row where skew is not 0).

The multisets of lengths and loads belong to the case, so its work does not
depend on the seed; the seed draws every value, the order of the events and
which expert has which load.
"""

from __future__ import annotations

import math
from typing import Dict, List, Optional

import torch

own = False

EPS = 1e-6
_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _case(name, op, mode, dtype, batch, length, lens, **more):
    case = {"op": op, "mode": mode, "dtype": dtype, "batch": batch, "length": length, "lens": lens, **more}
    if name:
        case["name"] = name
    return case


def listed() -> List[Dict]:
    return [
        # One event between two layers of an event-by-event reconstruction: the
        # smallest call, all latency.
        _case("rms_event_fwd", "rms", "fwd", "bf16", 1, 187, "packed", dim=384, residual=True, params="f32"),
        # The headline training batch (256 events of up to 768 pulses, 12 heads
        # of 32): the norm of every sub-layer, with its residual sum.
        _case("rms_padded_step", "rms", "step", "bf16", 256, 768, "uniform", dim=384, residual=True, params="f32"),
        # A summary token per event through a trained block, a few at a time.
        _case("rms8_token_fwd", "rms8", "fwd", "bf16", 1, 4, "packed", dim=768, residual=True, params="bf16"),
        # A large packed batch of a wide model in half precision.
        _case("rms8_wide_fwd", "rms8", "fwd", "f16", 1, 65536, "packed", dim=1024, residual=True, params="f16"),
        # The same few tokens between a block's router and its experts.
        _case("route_token_fwd", "route", "fwd", "f32", 1, 4, "packed", experts=8, top=2, softmax="chosen"),
        # The headline batch in a model of many small experts.
        _case("route_padded_step", "route", "step", "f32", 256, 768, "uniform", experts=64, top=4, softmax="chosen"),
        # One event's rows to eight experts and back.
        _case("shuffle_event_fwd", "shuffle", "fwd", "bf16", 1, 187, "packed", dim=384, experts=8, top=2),
        # The headline batch's, in a training step.
        _case("shuffle_padded_step", "shuffle", "step", "bf16", 256, 768, "uniform", dim=384, experts=16, top=2),
        # Few tokens through a trained model's experts: their weights are what is read.
        _case("experts_token_fwd", "experts", "fwd", "bf16", 1, 4, "packed", dim=768, hidden=2048, act="silu", experts=8,
              top=2, skew=0.9),
        # The headline training step: two experts a token, of 16 at half the
        # width of its feed-forward.
        _case("experts_padded_step", "experts", "step", "bf16", 256, 768, "uniform", dim=384, hidden=512, act="silu",
              experts=16, top=2, skew=0.5),
        # A step on a large packed batch of a wide model with many experts.
        _case("experts_wide_step", "experts", "step", "bf16", 1, 32768, "packed", dim=1024, hidden=1376, act="silu",
              experts=32, top=2, skew=0.5),
        # The wide-head configuration (8 heads of 64) in float32, one expert a token.
        _case("experts_step_f32", "experts", "step", "f32", 4, 4096, "full", dim=512, hidden=704, act="gelu", experts=8,
              top=1, skew=0.5),
    ]


def _logint(rng, lo, hi) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(case) -> float:
    """Seconds of a pass at rough rates, to hold drawn cases to the listed ones."""
    w = work(case)
    return w["bytes"] / 4e12 + w["flops"] / (1e14 if case["dtype"] == "f32" else 6e14)


def draw(rng) -> Dict:
    op = rng.choice(["rms", "rms8", "route", "shuffle", "shuffle", "experts", "experts", "experts"])
    top = max(_cost(c) for c in listed() if c["op"] == op)
    while True:
        mode = "fwd" if op == "rms8" else rng.choice(["fwd", "step", "step"])
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        batch = _logint(rng, 1, 512)
        length = _logint(rng, 1, 4096)
        lens = rng.choice(["packed", "uniform", "uniform", "full"])
        if batch * length > 250_000:
            continue
        more = {}
        if op in ("route", "shuffle", "experts"):
            more["experts"] = _logint(rng, 2, 256 if op == "route" else 64)
            more["top"] = min(more["experts"], rng.choice([1, 2, 2, 3, 4, 8]))
        if op in ("rms", "rms8", "shuffle"):
            more["dim"] = _logint(rng, 8, 8192)
        if op in ("rms", "rms8"):
            more.update(residual=rng.random() < 0.5, params=rng.choice(["f32", dtype]))
        elif op == "route":
            more["softmax"] = rng.choice(["chosen", "all"])
        elif op == "experts":
            more.update(dim=8 * _logint(rng, 4, 160), hidden=8 * _logint(rng, 8, 256),
                        act=rng.choice(["silu", "gelu", "gelu_tanh"]), skew=rng.choice([0.0, 0.5, 0.9]))
        case = _case("", op, mode, dtype, batch, length, lens, **more)
        if _cost(case) <= top:
            return case


def _lengths(case) -> Optional[List[int]]:
    """The events' lengths (the order is drawn with the inputs), or None where every row is a token."""
    b, top = case["batch"], case["length"]
    if case["lens"] != "uniform":
        return None
    lo = min(16, top)
    return [lo + int((top + 1 - lo) * (i + 0.5) / b) for i in range(b)]


def _tokens(case) -> int:
    lens = _lengths(case)
    return case["batch"] * case["length"] if lens is None else sum(lens)


def _loads(case) -> List[int]:
    """Rows of each expert (which one has which is drawn with the inputs)."""
    e, rows = case["experts"], _tokens(case) * case["top"]
    share = [1.0 + case["skew"] * (2.0 * (i + 0.5) / e - 1.0) for i in range(e)]
    if case["skew"] and e > 4:
        share[0] = 0.0
    ends = [sum(share[: i + 1]) / sum(share) for i in range(e)]
    ends = [0] + [int(round(rows * x)) for x in ends]
    return [b - a for a, b in zip(ends, ends[1:])]


def _lead(case):
    return (case["batch"] * case["length"],) if case["lens"] == "packed" else (case["batch"], case["length"])


def _sorted_slots(experts, n):
    """(order, place, offsets) of the slots by expert: a stable sort, slots of no expert (-1) last."""
    ids = torch.where(experts < 0, n, experts).reshape(-1).long()
    ids, order = torch.sort(ids, stable=True)
    offsets = torch.searchsorted(ids, torch.arange(n + 1, device=ids.device))
    rows = torch.arange(ids.numel(), device=ids.device)
    none = ids == n
    place = torch.empty_like(rows)
    place[order] = torch.where(none, -1, rows)
    order = torch.where(none, -1, order)
    return order.int(), place.reshape(experts.shape).int(), offsets.int()


def _inputs(case, seed: int) -> Dict[str, torch.Tensor]:
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    op, dt, lead, step = case["op"], _TYPES[case["dtype"]], _lead(case), case["mode"] == "step"

    def rn(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    x: Dict[str, torch.Tensor] = {}
    lens = _lengths(case)
    if lens is not None:
        order = torch.randperm(len(lens), generator=host)
        x["lens"] = torch.tensor(lens, dtype=torch.int32)[order].to(dev)
    if op in ("rms", "rms8"):
        dim = case["dim"]
        # A residual stream: channels with offsets and scales of their own.
        x["x"] = (rn(*lead, dim) * (0.5 + rn(dim).abs()) + 0.5 * rn(dim)).to(dt)
        if case["residual"]:
            x["r"] = (2.0 * rn(*lead, dim) + rn(dim)).to(dt)
        x["w"] = (1.0 + 0.2 * rn(dim)).to(_TYPES[case["params"]])
        if step:
            x["dy"] = (0.01 * rn(*lead, dim)).to(dt)
            if case["residual"]:
                x["ds"] = (0.01 * rn(*lead, dim)).to(dt)
        return x
    n, top = case["experts"], case["top"]
    if op == "route":
        # A router's logits, with a preference of its own for some experts.
        x["logits"] = (1.5 * rn(*lead, n) + 0.5 * rn(n)).to(dt)
        if step:
            x["dw"] = 0.1 * rn(*lead, top)
    elif op == "shuffle":
        dim, rows = case["dim"], math.prod(lead) * top
        chosen = torch.argsort(1.5 * rn(*lead, n) + 0.5 * rn(n), dim=-1, descending=True)[..., :top].int()
        pad = _padding(case, x)
        if pad is not None:
            chosen = chosen.masked_fill(pad, -1)
        x["order"], x["place"], x["offsets"] = _sorted_slots(chosen, n)
        w = torch.softmax(1.5 * rn(*lead, top), dim=-1)
        x["w"] = w if pad is None else w.masked_fill(pad, 0.0)
        x["x"] = rn(*lead, dim).to(dt)
        x["ys"] = rn(rows, dim).to(dt)
        if step:
            x["dxs"] = (0.05 * rn(rows, dim)).to(dt)
            x["dy"] = (0.05 * rn(*lead, dim)).to(dt)
    else:
        dim, hidden, rows = case["dim"], case["hidden"], math.prod(lead) * top
        loads = torch.tensor(_loads(case))[torch.randperm(n, generator=host)]
        x["offsets"] = torch.cat([loads.new_zeros(1), loads.cumsum(0)]).int().to(dev)
        # What a norm hands the block, and weights at the usual scale.
        x["x"] = rn(rows, dim).to(dt)
        x["wg"] = (rn(n, hidden, dim) / dim ** 0.5).to(dt)
        x["wu"] = (rn(n, hidden, dim) / dim ** 0.5).to(dt)
        x["wd"] = (rn(n, dim, hidden) / hidden ** 0.5).to(dt)
        if step:
            x["dy"] = (0.05 * rn(rows, dim)).to(dt)
    return x


_LEAVES = {"rms": ("x", "r", "w"), "rms8": (), "route": ("logits",), "shuffle": ("x", "ys", "w"),
           "experts": ("x", "wg", "wu", "wd")}


def prepare(case, seed: int) -> Dict:
    x = _inputs(case, seed)
    if own and case["mode"] == "step":
        for name in _LEAVES[case["op"]]:
            if name in x:
                x[name].requires_grad_(True)
    return {"case": case, "x": x}


def run(state):
    """One forward, or one forward and backward: the outputs, then the
    gradients of the rows (and the residual) and of the weights."""
    case, x = state["case"], state["x"]
    if own:
        return _own(case, x)
    return {"rms": _plain_rms, "rms8": _plain_rms, "route": _plain_route, "shuffle": _plain_shuffle,
            "experts": _plain_experts}[case["op"]](case, x)


def _own(case, x):
    import flash_spacetime_amd as fst

    op, step = case["op"], case["mode"] == "step"
    if op == "rms8":
        return list(fst.flash_rms_norm_fp8(x["x"], x["w"], EPS, residual=x.get("r"), seqlens=x.get("lens")))
    more = []
    if op == "rms":
        out = fst.flash_rms_norm(x["x"], x["w"], EPS, residual=x.get("r"), seqlens=x.get("lens"))
        outs, dys = (list(out), ["dy", "ds"]) if case["residual"] else ([out], ["dy"])
    elif op == "route":
        weights, experts = fst.flash_expert_route(x["logits"], case["top"], normalize=case["softmax"] == "chosen",
                                                  seqlens=x.get("lens"))
        outs, dys = [weights], ["dw"]
        more = [experts, *fst.flash_expert_sort(experts, case["experts"])]
    elif op == "shuffle":
        order = fst.ExpertOrder(x["order"], x["place"], x["offsets"])
        outs = [fst.flash_expert_dispatch(x["x"], order), fst.flash_expert_combine(x["ys"], x["w"], order)]
        dys = ["dxs", "dy"]
    else:
        outs = [fst.flash_expert_feed_forward(x["x"], x["offsets"], x["wg"], x["wu"], x["wd"], case["act"])]
        dys = ["dy"]
    if not step:
        return outs + more
    grads = torch.autograd.grad(outs, [x[n] for n in _LEAVES[op] if n in x], [x[n] for n in dys])
    return [o.detach() for o in outs] + more + list(grads)


def _padding(case, x) -> Optional[torch.Tensor]:
    """[batch, length, 1], true past the events' lengths; None without lengths."""
    if "lens" not in x:
        return None
    return (torch.arange(case["length"], device=x["lens"].device)[None, :] >= x["lens"][:, None])[..., None]


def _plain_rms(case, x):
    dt, pad = x["x"].dtype, _padding(case, x)

    def rows(t):
        t = t.float()
        return t if pad is None else t.masked_fill(pad, 0.0)

    s = rows(x["x"])
    if case["residual"]:
        s = (s + rows(x["r"])).to(dt).float()
    w = x["w"].float()
    rstd = (s.square().mean(-1, keepdim=True) + EPS).rsqrt()
    xhat = s * rstd
    y = xhat * w
    sums = [s.to(dt)] if case["residual"] else []
    if case["op"] == "rms8":
        scale = (y.abs().amax(-1, keepdim=True) / 448.0).clamp(min=2.0 ** -126)
        q = (y / scale).to(torch.float8_e4m3fn)
        return [q, rows(scale)[..., 0]] + sums
    outs = [y.to(dt)] + sums
    if case["mode"] == "fwd":
        return outs
    dy = rows(x["dy"])
    g = dy * w
    dx = rstd * (g - xhat * (g * xhat).mean(-1, keepdim=True))
    if case["residual"]:
        dx = dx + rows(x["ds"])
    dw = (dy * xhat).sum(tuple(range(dx.dim() - 1)))
    dx = dx.to(dt)
    return outs + ([dx, dx.clone()] if case["residual"] else [dx]) + [dw.to(x["w"].dtype)]


def _plain_route(case, x):
    n, top, pad = case["experts"], case["top"], _padding(case, x)
    logits = x["logits"].float()
    best, at = torch.sort(logits, dim=-1, descending=True, stable=True)
    best, at = best[..., :top], at[..., :top]
    e = torch.exp(best - best[..., :1])
    if case["softmax"] == "chosen":
        weights = e / e.sum(-1, keepdim=True)
    else:
        weights = e / torch.exp(logits - best[..., :1]).sum(-1, keepdim=True)
    experts = at.int()
    if pad is not None:
        weights, experts = weights.masked_fill(pad, 0.0), experts.masked_fill(pad, -1)
    outs = [weights, experts, *_sorted_slots(experts, n)]
    if case["mode"] == "fwd":
        return outs
    dw = x["dw"] if pad is None else x["dw"].masked_fill(pad, 0.0)
    mean = (weights * dw).sum(-1, keepdim=True)
    if case["softmax"] == "chosen":
        grad = torch.zeros_like(logits).scatter(-1, at, weights * (dw - mean))
    else:
        p = torch.exp(logits - best[..., :1])
        grad = (-mean * p / p.sum(-1, keepdim=True)).scatter_add(-1, at, weights * dw)
    return outs + [grad.to(x["logits"].dtype)]


def _plain_shuffle(case, x):
    dt, dim, place = x["x"].dtype, case["dim"], x["place"].long()
    lead, top, rows = place.shape[:-1], case["top"], place.numel()
    # Slots of no expert read and write one row more, which is dropped.
    at = torch.where(place < 0, rows, place).reshape(-1)

    def spread(t):
        t = t[..., None, :].expand(*lead, top, dim).reshape(rows, dim)
        return torch.zeros(rows + 1, dim, device=t.device, dtype=t.dtype).index_copy(0, at, t)[:rows]

    def gathered(t):
        return torch.cat([t.float(), torch.zeros(1, dim, device=t.device)])[at].reshape(*lead, top, dim)

    w = x["w"][..., None]
    xs = spread(x["x"])
    ys = gathered(x["ys"])
    outs = [xs, (w * ys).sum(-2).to(dt)]
    if case["mode"] == "fwd":
        return outs
    dx = gathered(x["dxs"]).sum(-2).to(dt)
    dy = x["dy"].float()[..., None, :]
    dys = torch.zeros(rows + 1, dim, device=dy.device).index_copy(0, at, (w * dy).reshape(rows, dim))[:rows].to(dt)
    return outs + [dx, dys, (dy * ys).sum(-1)]


def _plain_experts(case, x):
    """Every expert's rows as one [cap, dim] of a batch of products."""
    dt, n, dim, hidden, cap = x["x"].dtype, case["experts"], case["dim"], case["hidden"], max(max(_loads(case)), 1)
    rows = x["x"].shape[0]
    offsets = x["offsets"].long()
    at = offsets[:-1, None] + torch.arange(cap, device=offsets.device)
    at = torch.where(at < offsets[1:, None], at, rows)  # past an expert's last: a row of zeros

    def batched(t):
        return torch.cat([t.float(), torch.zeros(1, dim, device=t.device)])[at.reshape(-1)].reshape(n, cap, dim)

    def back(t):
        full = torch.zeros(rows + 1, dim, device=t.device)
        return full.index_copy(0, at.reshape(-1), t.reshape(-1, dim))[:rows].to(dt)

    def turned(t):
        return t.transpose(1, 2).contiguous()

    xs, wg, wu, wd = batched(x["x"]), x["wg"].float(), x["wu"].float(), x["wd"].float()
    a, u = torch.bmm(xs, turned(wg)), torch.bmm(xs, turned(wu))
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
    outs = [back(torch.bmm(h, turned(wd)))]
    if case["mode"] == "fwd":
        return outs
    dy = batched(x["dy"])
    dh = torch.bmm(dy, wd)
    if case["act"] == "silu":
        slope = gate * (1.0 + a * (1.0 - gate))
    elif case["act"] == "gelu":
        slope = gate + a * torch.exp(-0.5 * a * a) * (2.0 * math.pi) ** -0.5
    else:
        slope = 0.5 * (1.0 + t) + 0.5 * a * (1.0 - t * t) * (2.0 / math.pi) ** 0.5 * (1.0 + 3 * 0.044715 * a * a)
    da, du = dh * u * slope, dh * act
    outs.append(back(torch.bmm(da, wg) + torch.bmm(du, wu)))
    return outs + [torch.bmm(turned(da), xs).to(dt), torch.bmm(turned(du), xs).to(dt), torch.bmm(turned(dy), h).to(dt)]


def work(case) -> Dict[str, float]:
    """Each valid row read once, every row of the outputs written once (rows of
    padding and of no expert are zeros the operators write), and the definition's
    operations over the valid rows."""
    rows, valid = case["batch"] * case["length"], _tokens(case)
    es, step, op = 4 if case["dtype"] == "f32" else 2, case["mode"] == "step", case["op"]
    if op in ("rms", "rms8"):
        dim, wide = case["dim"], 2 if case["residual"] else 1
        ps = 4 if case["params"] == "f32" else 2
        nbytes = dim * es * (wide * valid + (wide - 1) * rows) + dim * ps
        nbytes += rows * (dim + 4) if op == "rms8" else dim * es * rows
        flops = (wide + 3 if op == "rms" else wide + 5) * valid * dim
        if step:
            # dy and ds in; one dx (the residual's gradient is the same) and dw out.
            nbytes += dim * es * (wide * valid + rows) + dim * ps
            flops += (8 + wide) * valid * dim
        return {"bytes": float(nbytes), "flops": float(flops)}
    n, top = case["experts"], case["top"]
    slots, used = rows * top, valid * top
    if op == "route":
        # Logits in; weights, experts, order and place out.
        nbytes = es * valid * n + 16 * slots + 4 * (n + 1)
        flops = valid * n * (top + 3)
        if step:
            nbytes += 4 * used + es * rows * n
            flops += 4 * used + (4 * valid * n if case["softmax"] == "all" else 0)
        return {"bytes": float(nbytes), "flops": float(flops)}
    dim = case["dim"]
    if op == "shuffle":
        nbytes = dim * es * (valid + slots + used + rows) + 8 * slots
        flops = 2 * used * dim
        if step:
            nbytes += dim * es * (used + rows + valid + slots) + 4 * slots
            flops += 4 * used * dim
        return {"bytes": float(nbytes), "flops": float(flops)}
    hidden = case["hidden"]
    busy = sum(1 for v in _loads(case) if v)
    nbytes = es * (dim * (used + slots) + 3 * busy * dim * hidden) + 4 * (n + 1)
    flops = 6.0 * used * dim * hidden
    if step:
        nbytes += es * (dim * (used + slots) + 3 * n * dim * hidden)
        flops += 12.0 * used * dim * hidden
    return {"bytes": float(nbytes), "flops": flops}


# ---------------------------------------------------------------------------
# The same results in 64 bits, from the definitions: the valid rows gathered,
# the gradients by differentiating the definition, the rows put back.
# ---------------------------------------------------------------------------


def exact(case, seed: int) -> Optional[List[torch.Tensor]]:
    x = _inputs(case, seed)
    step, op, lead = case["mode"] == "step", case["op"], _lead(case)
    dev = next(iter(x.values())).device
    valid = torch.ones(lead, dtype=torch.bool, device=dev)
    if "lens" in x:
        for i, n in enumerate(x["lens"].tolist()):
            valid[i, n:] = False

    def back(t):
        full = torch.zeros(*lead, *t.shape[1:], dtype=torch.float64, device=dev)
        full[valid] = t.detach()
        return full

    def leaf(t):
        return t.double().requires_grad_(step)

    if op in ("rms", "rms8"):
        s = x["x"][valid]
        if case["residual"]:
            s = (s.float() + x["r"][valid].float()).to(s.dtype)
        s, w = leaf(s), leaf(x["w"])
        y = s / torch.sqrt((s * s).sum(-1, keepdim=True) / case["dim"] + EPS) * w
        sums = [back(s)] if case["residual"] else []
        if op == "rms8":
            top = y.abs().max(-1).values
            # what the 8 bits and their scale stand for, before they are rounded
            return [back(y * (448.0 / torch.where(top > 0, top, 1.0))[:, None]), back(top / 448.0)] + sums
        outs = [back(y)] + sums
        if not step:
            return outs
        ds, dw = torch.autograd.grad(y, (s, w), x["dy"][valid].double())
        if case["residual"]:
            ds = ds + x["ds"][valid].double()
        ds = back(ds)
        return outs + ([ds, ds.clone()] if case["residual"] else [ds]) + [dw]

    if op == "route":
        logits = leaf(x["logits"][valid])
        at = torch.sort(-logits.detach(), dim=-1, stable=True).indices[:, : case["top"]]
        if case["softmax"] == "chosen":
            weights = torch.softmax(torch.gather(logits, 1, at), dim=1)
        else:
            weights = torch.gather(torch.softmax(logits, dim=1), 1, at)
        outs = [back(weights), None, None, None, None]
        if not step:
            return outs
        return outs + [back(torch.autograd.grad(weights, logits, x["dw"][valid].double())[0])]

    if op == "shuffle":
        # Row r of the experts' order holds token order[r] // top, in slot order[r] % top.
        dim, top, tokens = case["dim"], case["top"], math.prod(lead)
        used = int(x["offsets"][-1])
        slot = x["order"][:used].long()
        token = slot // top
        xs = torch.zeros(tokens * top, dim, dtype=torch.float64, device=dev)
        xs[:used] = x["x"].reshape(tokens, dim)[token].double()
        ys, w = x["ys"][:used].double(), x["w"].reshape(-1)[slot].double()[:, None]
        outs = [xs, torch.zeros(tokens, dim, dtype=torch.float64, device=dev).index_add(0, token, w * ys).reshape(*lead, dim)]
        if not step:
            return outs
        dx = torch.zeros(tokens, dim, dtype=torch.float64, device=dev).index_add(0, token, x["dxs"][:used].double())
        dy = x["dy"].reshape(tokens, dim)[token].double()
        dys = torch.zeros_like(xs)
        dys[:used] = w * dy
        dw = torch.zeros(tokens * top, dtype=torch.float64, device=dev)
        dw[slot] = (dy * ys).sum(-1)
        return outs + [dx.reshape(*lead, dim), dys, dw.reshape(*lead, top)]

    y = torch.zeros(x["x"].shape, dtype=torch.float64, device=dev)
    grads = [torch.zeros(x[name].shape, dtype=torch.float64, device=dev) for name in _LEAVES["experts"]]
    ends = x["offsets"].tolist()
    for e, (lo, hi) in enumerate(zip(ends, ends[1:])):
        rows, wg, wu, wd = leaf(x["x"][lo:hi]), leaf(x["wg"][e]), leaf(x["wu"][e]), leaf(x["wd"][e])
        gate = rows @ wg.t()
        if case["act"] == "silu":
            gate = gate / (1.0 + torch.exp(-gate))
        elif case["act"] == "gelu":
            gate = gate * torch.erfc(-gate / math.sqrt(2.0)) / 2.0
        else:
            # gelu_tanh: x sigmoid(2 z) = x (1 + tanh z) / 2
            gate = gate / (1.0 + torch.exp(-2.0 * math.sqrt(2.0 / math.pi) * (gate + 0.044715 * gate ** 3)))
        out = (gate * (rows @ wu.t())) @ wd.t()
        y[lo:hi] = out.detach()
        if step:
            got = torch.autograd.grad(out, (rows, wg, wu, wd), x["dy"][lo:hi].double())
            grads[0][lo:hi] = got[0]
            for full, g in zip(grads[1:], got[1:]):
                full[e] = g
    return [y] + (grads if step else [])
