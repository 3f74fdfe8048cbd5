"""GPU tests of SpacetimeBlock with root-mean-square norms and a mixture of experts,
against the block's definition in float64 on the CPU, and of those operators under
torch's other ways of running a call.

Tolerances as the block's own test (test_block_gpu.py). Experts are chosen by the
operator's logits, which the kernels' rounding moves: the definition is given the
choice that was made, so that it differentiates the same function.
"""

import copy

import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx
from torch.nn import functional as F

import oracle
from tests._cases import rel_err, seed_of

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from flash_spacetime_amd import (ExpertOrder, SpacetimeBlock, _lib, attention_rel_oracle_inputs, experts,
                                     flash_expert_combine, flash_expert_dispatch, flash_expert_feed_forward,
                                     flash_expert_route, flash_expert_sort, flash_rms_norm, flash_rms_norm_fp8, merge_heads)

DEV = "cuda"


def _reference(ref, x, feats, valid, chosen):
    mask = oracle.float_padding_mask(valid, torch.float64)
    q, k, v = attention_rel_oracle_inputs(ref.attn, ref.norm1(x), None)
    att = oracle.attention(q, k, v, feats, ref.attn.rel_proj.weight, ref.attn.rel_proj.bias, key_padding_mask=mask)
    x = x + ref.attn.proj(merge_heads(att))
    y = ref.norm2(x)
    if ref.experts is None:
        return x + ref.ffn_down(F.silu(ref.ffn_gate(y)) * ref.ffn_up(y))
    w = torch.softmax(torch.gather(ref.router(y), -1, chosen.clamp(min=0)), -1)
    for e in range(ref.experts):
        h = F.silu(y @ ref.experts_gate[e].t()) * (y @ ref.experts_up[e].t())
        x = x + (w * (chosen == e)).sum(-1, keepdim=True) * (h @ ref.experts_down[e].t())
    return x


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("mask", ["lengths", "holes", "packed"])
@pytest.mark.parametrize("norm,count", [("rms", None), ("rms", 6), ("layer", 3)])
def test_block_matches_its_definition(monkeypatch, dtype, mask, norm, count):
    batch, length, dim = 4, 40, 128
    gen = torch.Generator().manual_seed(seed_of("block", dtype, mask, norm, count))
    ref = SpacetimeBlock(dim, 4, norm=norm, experts=count, hidden=192, eps=1e-6, dtype=torch.float64)
    with torch.no_grad():
        for name, p in ref.named_parameters():
            v = torch.randn(p.shape, generator=gen, dtype=torch.float64) * (p.shape[-1] ** -0.5)
            p.copy_(1 + 0.1 * v if name in ("norm1.weight", "norm2.weight") else v)
    mod = copy.deepcopy(ref).to(DEV, dtype)
    with torch.no_grad():
        for p, r in zip(mod.parameters(), ref.parameters()):
            r.copy_(p.double().cpu())
    x64 = torch.randn(batch, length, dim, generator=gen, dtype=torch.float64).to(dtype).double()
    feats = torch.randn(batch, length, 5, generator=gen, dtype=torch.float64)
    if mask == "holes":
        valid = torch.rand(batch, length, generator=gen) < 0.6
        valid[:, 3] = True
    else:
        valid = torch.arange(length)[None, :] < torch.tensor([length, 17, 1, 30])[:, None]
    gw = torch.randn(batch, length, dim, generator=gen, dtype=torch.float64)
    made, route = [], experts.flash_expert_route

    def seen(*args, **kwargs):
        out = route(*args, **kwargs)
        made.append(out[1].cpu().long())
        return out

    monkeypatch.setattr(experts, "flash_expert_route", seen)
    pad = ~valid.to(DEV)
    x = x64.to(DEV, dtype)
    x[pad] = float("nan")  # what padding holds is nobody's business
    x.requires_grad_(True)
    if mask == "packed":
        cu = torch.tensor([0, *valid.sum(1).cumsum(0).tolist()], dtype=torch.int32, device=DEV)
        # events one after the other, then tokens of no event
        rows = torch.cat([x[~pad], torch.full((9, dim), float("nan"), device=DEV, dtype=dtype)])
        out = mod(rows, torch.cat([feats[valid], feats[0, :9]]).to(DEV), cu_seqlens=cu)
        assert bool((out[-9:] == 0).all())
        out = torch.zeros(batch, length, dim, device=DEV, dtype=dtype).index_put((~pad,), out[:-9])
    elif mask == "lengths":
        out = mod(x, feats.to(DEV), seqlens=valid.sum(1).to(DEV))
    else:
        out = mod(x, feats.to(DEV), key_padding_mask=pad)
    out.backward(gw.to(DEV, dtype))
    assert bool((out.detach()[pad] == 0).all()) and bool((x.grad[pad] == 0).all())

    chosen = None
    if count is not None:
        (got,) = made
        chosen = torch.full((batch, length, 2), -1)
        chosen[valid] = got[valid] if mask == "lengths" else got[: int(valid.sum())]
        assert bool((chosen[valid] >= 0).all())
    xr = x64.clone().requires_grad_(True)
    want = _reference(ref, xr, feats, valid, chosen)
    vm = valid[..., None].expand(want.shape)
    (want * (gw.to(dtype).double() * vm)).sum().backward()
    tol = 2e-2 if dtype == torch.bfloat16 else 2e-4
    gtol = 2e-2 if dtype == torch.bfloat16 else 1e-3
    assert rel_err(out.detach().double().cpu() * vm, want.detach() * vm) <= tol
    assert rel_err(x.grad.double().cpu(), xr.grad) <= gtol
    for (name, p), r in zip(mod.named_parameters(), ref.parameters()):
        err = rel_err(p.grad.double().cpu(), r.grad)
        assert err <= gtol, f"grad {name}: relative error {err:.3e}"


@pytest.mark.parametrize("shape", [(0, 7), (2, 0), (3, 5), (0,)], ids=["no_event", "no_length", "no_token", "packed"])
def test_batches_without_tokens(shape):
    blk = SpacetimeBlock(64, 2, norm="rms", experts=4, device=DEV, dtype=torch.bfloat16)
    x = torch.ones(*shape, 64, device=DEV, dtype=torch.bfloat16, requires_grad=True)
    feats = torch.ones(*shape, 4, device=DEV)
    if len(shape) == 1:
        y = blk(x, feats, cu_seqlens=torch.zeros(1, dtype=torch.int32, device=DEV))
    else:
        y = blk(x, feats, torch.zeros(shape[0], dtype=torch.int32, device=DEV))
    assert y.shape == x.shape and bool((y == 0).all())
    grads = torch.autograd.grad(y, [x, *blk.parameters()], torch.ones_like(y), allow_unused=True)
    for name, g in zip(["x", *(n for n, _ in blk.named_parameters())], grads):
        assert g is None or bool((g == 0).all()), name


@pytest.mark.parametrize("low", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
def test_block_under_autocast(low):
    """float32 parameters and stream: the output and every gradient are float32 and finite,
    those of the float32 block up to a 16-bit block's roundings where the choice of
    experts is the same (one expert: the mixture is a feed-forward)."""
    gen = torch.Generator().manual_seed(5)
    x, feats, dy = (torch.randn(3, 24, n, generator=gen).to(DEV) for n in (64, 4, 64))
    lens = torch.tensor([24, 7, 15], device=DEV)

    def run(blk):
        leaf = x.clone().requires_grad_(True)
        y = blk(leaf, feats, lens)
        return [y.detach(), *torch.autograd.grad(y, [leaf, *blk.parameters()], dy.to(y.dtype), allow_unused=True)]

    for count, top_k in ((1, 1), (5, 2)):
        blk = SpacetimeBlock(64, 4, norm="rms", experts=count, top_k=top_k, device=DEV)
        want = run(blk)
        with torch.autocast("cuda", dtype=low):
            got = run(blk)
        for a, b in zip(got, want):
            assert a.dtype == torch.float32 and bool(a.isfinite().all())
            if count == 1:
                assert float((a - b).double().norm()) <= 2e-2 * float(b.double().norm()) + 1e-6


def _calls():
    """Every operator's call as a function of its floating tensors, and those."""
    gen = torch.Generator().manual_seed(11)
    rn = lambda *s: torch.randn(*s, generator=gen).to(DEV)  # noqa: E731
    x, r, w, logits = rn(50, 64), rn(50, 64), rn(64), rn(50, 6)
    order = flash_expert_sort(flash_expert_route(logits, 2)[1], 6)
    wg, wu, wd = rn(6, 128, 64) / 8, rn(6, 128, 64) / 8, rn(6, 64, 128) / 11
    return {
        "rms": (lambda x, w: flash_rms_norm(x, w), [x, w]),
        "rms_residual": (lambda x, r, w: sum(flash_rms_norm(x, w, residual=r)), [x, r, w]),
        "route": (lambda t: flash_expert_route(t, 2)[0], [logits]),
        "route_all": (lambda t: flash_expert_route(t, 2, normalize=False)[0], [logits]),
        "dispatch": (lambda x: flash_expert_dispatch(x, order), [x]),
        "combine": (lambda y, w: flash_expert_combine(y, w, order), [rn(100, 64), rn(50, 2)]),
        "ffn": (lambda x, *t: flash_expert_feed_forward(x, order.offsets, *t), [rn(100, 64), wg, wu, wd]),
    }


NAMES = ["rms", "rms_residual", "route", "route_all", "dispatch", "combine", "ffn"]


def _leave_nan(*shapes):
    for _ in range(2):
        _ = [torch.full(s, float("nan"), device=DEV) for s in shapes for _ in range(4)]


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name", NAMES)
def test_traced_calls_compute(name, grad):
    f, tensors = _calls()[name]
    traced = torch.jit.trace(f, tuple(t.clone().requires_grad_(grad) for t in tensors), check_trace=False)
    other = [1.5 * t.flip(0) for t in tensors]
    want = f(*other)
    _leave_nan(want.shape)
    assert torch.equal(traced(*other), want)


def test_traced_8_bits_and_block_compute():
    x, w = _calls()["rms"][1]
    traced = torch.jit.trace(lambda x, w: tuple(flash_rms_norm_fp8(x, w)), (x, w), check_trace=False)
    got, want = traced(2 * x.flip(0), w), flash_rms_norm_fp8(2 * x.flip(0), w)
    assert all(torch.equal(a.float(), b.float()) for a, b in zip(got, want))
    blk = SpacetimeBlock(64, 4, norm="rms", experts=4, device=DEV)
    gen = torch.Generator().manual_seed(2)
    x, feats = torch.randn(2, 20, 64, generator=gen).to(DEV), torch.randn(2, 20, 4, generator=gen).to(DEV)
    lens = torch.tensor([20, 7], device=DEV)
    traced = torch.jit.trace(blk, (x, feats, lens), check_trace=False)
    other = 1.5 * x.flip(1)
    want = blk(other, feats, lens)
    _leave_nan(want.shape, (80, 64), (80, 192))
    assert torch.equal(traced(other, feats, lens), want)


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_derivatives_are_refused(name, grad):
    f, tensors = _calls()[name]
    for i, t in enumerate(tensors):
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(t.clone().requires_grad_(grad), torch.ones_like(t))
            with pytest.raises(NotImplementedError, match="jvp"):
                f(*tensors[:i], dual, *tensors[i + 1:])
    f(*tensors)


@pytest.mark.parametrize("name", NAMES)
def test_make_fx_is_refused(monkeypatch, name):
    f, tensors = _calls()[name]
    for host in (True, False):
        with monkeypatch.context() as m:
            if not host:
                m.setattr(_lib, "host", lambda: None)
            with pytest.raises(RuntimeError, match="make_fx"):
                make_fx(f)(*tensors)
            leaf = tensors[0].clone().requires_grad_(True)
            y = f(leaf, *tensors[1:])
            with pytest.raises(RuntimeError, match="make_fx"):
                make_fx(lambda g: torch.autograd.grad(y, leaf, g, retain_graph=True))(torch.ones_like(y))
            torch.autograd.grad(y, leaf, torch.ones_like(y))


@pytest.mark.parametrize("name", NAMES)
def test_only_first_derivatives_and_unchanged_inputs(monkeypatch, name):
    """A second derivative raises, and so does a tensor kept for the backward that was
    changed in place since, with the host extension as without it."""
    f, tensors = _calls()[name]
    for host in (True, False):
        with monkeypatch.context() as m:
            if not host:
                m.setattr(_lib, "host", lambda: None)
            leaves = [t.clone().requires_grad_(True) for t in tensors]
            g = torch.autograd.grad(f(*leaves).square().sum(), leaves[0], create_graph=True)[0]
            with pytest.raises(RuntimeError, match="twice|once_differentiable"):
                g.sum().backward()
            if name in ("rms", "route_all", "combine", "ffn"):
                leaves = [t.clone().requires_grad_(True) for t in tensors]
                y = f(*leaves)
                leaves[0].detach().add_(1)
                with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                    y.sum().backward()


@pytest.mark.parametrize("name", NAMES)
def test_host_extension_and_python_path_agree(monkeypatch, name):
    """Bitwise, outputs and gradients; a kept graph runs twice; tensors of another stream."""
    f, tensors = _calls()[name]

    def run():
        leaves = [t.clone().requires_grad_(True) for t in tensors]
        y = f(*leaves)
        gen = torch.Generator(device=DEV).manual_seed(1)
        dy = torch.randn(y.shape, generator=gen, device=DEV)
        one = torch.autograd.grad(y, leaves, dy, retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(one, torch.autograd.grad(y, leaves, dy)))
        return [y.detach(), *one]

    want = run()
    with monkeypatch.context() as m:
        m.setattr(_lib, "host", lambda: None)
        assert all(torch.equal(a, b) for a, b in zip(run(), want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals():
    x, logits = torch.randn(6, 32, device=DEV), torch.randn(6, 4, device=DEV)
    ids = torch.zeros(6, 2, dtype=torch.int32, device=DEV)
    order = flash_expert_sort(ids, 4)
    ws = [torch.randn(*s, device=DEV) for s in ((4, 16, 32), (4, 16, 32), (4, 32, 16))]
    rows = torch.randn(12, 32, device=DEV)
    bad = [
        ("top_k", lambda: flash_expert_route(logits, 5)), ("top_k", lambda: flash_expert_route(logits, 0)),
        ("top_k", lambda: flash_expert_route(logits, True)), ("top_k", lambda: flash_expert_route(logits, 2.0)),
        ("16", lambda: flash_expert_route(torch.randn(3, 40, device=DEV), 17)),
        ("512", lambda: flash_expert_route(torch.randn(3, 513, device=DEV), 2)),
        ("bfloat16", lambda: flash_expert_route(logits.double(), 2)),
        ("seqlens", lambda: flash_expert_route(logits, 2, seqlens=torch.tensor([1, 2], device=DEV))),
        ("integer", lambda: flash_expert_sort(ids.float(), 4)), ("num_experts", lambda: flash_expert_sort(ids, 0)),
        ("num_experts", lambda: flash_expert_sort(ids, 2.0)), ("512", lambda: flash_expert_sort(ids, 513)),
        ("scalar", lambda: flash_expert_sort(ids[0, 0], 4)),
        ("ExpertOrder", lambda: flash_expert_dispatch(x, tuple(order))),
        ("place", lambda: flash_expert_dispatch(x, ExpertOrder(order.order, order.place.long(), order.offsets))),
        ("order.place", lambda: flash_expert_dispatch(x[:4], order)),
        ("on cuda", lambda: flash_expert_dispatch(x, ExpertOrder(order.order, order.place.cpu(), order.offsets))),
        ("offsets", lambda: flash_expert_combine(rows, torch.rand(6, 2, device=DEV),
                                                 ExpertOrder(order.order, order.place, order.offsets[:1]))),
        ("weights", lambda: flash_expert_combine(rows, torch.rand(6, 3, device=DEV), order)),
        ("weights", lambda: flash_expert_combine(rows, torch.rand(6, 2, device=DEV).half(), order)),
        ("ys must", lambda: flash_expert_combine(rows[None], torch.rand(6, 2, device=DEV), order)),
        ("activation", lambda: flash_expert_feed_forward(rows, order.offsets, *ws, "relu")),
        ("x must", lambda: flash_expert_feed_forward(rows[None], order.offsets, *ws)),
        ("w_gate", lambda: flash_expert_feed_forward(rows, order.offsets, ws[2], *ws[1:])),
        ("w_up", lambda: flash_expert_feed_forward(rows, order.offsets, ws[0], ws[1][:2], ws[2])),
        ("w_down", lambda: flash_expert_feed_forward(rows, order.offsets, ws[0], ws[1], ws[1])),
        ("dtype", lambda: flash_expert_feed_forward(rows, order.offsets, ws[0].half(), *ws[1:])),
        ("offsets", lambda: flash_expert_feed_forward(rows, order.offsets[:3], *ws)),
        ("offsets", lambda: flash_expert_feed_forward(rows, order.offsets.long(), *ws)),
        ("multiples of 8", lambda: flash_expert_feed_forward(rows[:, :30], order.offsets, ws[0][..., :30], ws[1][..., :30],
                                                             ws[2][:, :30])),
    ]
    for what, call in bad:
        with pytest.raises(ValueError, match=what):
            call()
    with pytest.raises(RuntimeError, match="GPU"):
        flash_expert_feed_forward(rows, order.offsets, ws[0].cpu(), *ws[1:])


@pytest.mark.parametrize("rc", [-1, -2, -3, -4])
@pytest.mark.parametrize("entry,name", [("fst_rms_norm_forward", "rms"), ("fst_expert_route", "route"),
                                        ("fst_expert_spread", "dispatch"), ("fst_expert_gather", "combine"),
                                        ("fst_expert_ffn_forward", "ffn")])
def test_failed_calls_raise(monkeypatch, entry, name, rc):
    """On the Python path: what the library refuses is a ValueError, any other failure a
    RuntimeError, and nothing is returned."""
    f, tensors = _calls()[name]
    lib = _lib.load()

    class Failing:
        def __getattr__(self, n):
            return (lambda *a: rc) if n == entry else getattr(lib, n)

    monkeypatch.setattr(_lib, "host", lambda: None)
    monkeypatch.setattr(_lib, "load", lambda: Failing())
    with pytest.raises(ValueError if rc in (-1, -2) else RuntimeError):
        f(*tensors)
