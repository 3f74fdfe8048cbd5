"""GPU tests of the layer norm, the feed-forward block and SpacetimeBlock under
torch's other ways of running a call: recorded, with forward-mode derivatives,
under autocast."""

import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

from tests._cases import seed_of

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from flash_spacetime_amd import (SpacetimeBlock, flash_gated_feed_forward, flash_layer_norm,
                                     flash_spacetime_attention, flash_spacetime_attention_qkv)

DEV = "cuda"


def _randn(key, *shapes):
    gen = torch.Generator().manual_seed(seed_of("modes", key))
    return [torch.randn(*s, generator=gen).to(DEV) for s in shapes]


def _calls():
    """Both operators' calls: a function of its tensors, and those."""
    x, r, w, b = _randn("norm", (50, 64), (50, 64), (64,), (64,))
    wg, wu, wd = _randn("ffn", (128, 64), (128, 64), (64, 128))
    return {
        "norm": (lambda x, w, b: flash_layer_norm(x, w, b), [x, w, b]),
        "norm_residual": (lambda x, r, w: sum(flash_layer_norm(x, w, residual=r)), [x, r, w]),
        "ffn": (lambda *t: flash_gated_feed_forward(*t), [x, wg / 8, wu / 8, wd / 11]),
    }


def _leave_nan(*shapes):
    """Memory of these shapes, freed, that holds NaN: what an output left unwritten shows."""
    for _ in range(2):
        _ = [torch.full(s, float("nan"), device=DEV) for s in shapes for _ in range(4)]


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name", ["norm", "norm_residual", "ffn"])
def test_traced_calls_compute(name, grad):
    """torch.jit.trace records the operator as a call, also beside the host extension:
    the traced function gives the operator's bits for inputs it has not seen."""
    f, tensors = _calls()[name]
    traced = torch.jit.trace(f, tuple(t.clone().requires_grad_(grad) for t in tensors), check_trace=False)
    other = [1.5 * t.flip(0) for t in tensors]
    want = f(*other)
    _leave_nan(want.shape)
    assert torch.equal(traced(*other), want)


def test_traced_block_computes():
    blk = SpacetimeBlock(64, 4, device=DEV)
    x, feats = _randn("block", (2, 20, 64), (2, 20, 4))
    lens = torch.tensor([20, 7], device=DEV)
    traced = torch.jit.trace(blk, (x, feats, lens), check_trace=False)
    other = 1.5 * x.flip(1)
    want = blk(other, feats, lens)
    _leave_nan(want.shape, (2, 20, 192))
    assert torch.equal(traced(other, feats, lens), want)


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name", ["norm", "norm_residual", "ffn"])
def test_forward_mode_derivatives_are_refused(name, grad):
    """They are not offered: a dual tensor in any place raises, with the host
    extension as without it, and is not taken for a constant."""
    f, tensors = _calls()[name]
    for i, t in enumerate(tensors):
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(t.clone().requires_grad_(grad), torch.ones_like(t))
            with pytest.raises(NotImplementedError, match="jvp"):
                f(*tensors[:i], dual, *tensors[i + 1:])
    f(*tensors)


@pytest.mark.parametrize("name", ["norm", "norm_residual", "ffn", "attention", "attention_qkv"])
def test_make_fx_is_refused(monkeypatch, name):
    """make_fx would record the outputs' allocation and not the launch: it is
    refused, forward and backward, with the host extension and without."""
    from flash_spacetime_amd import _lib

    if name.startswith("attention"):
        q, feats, w = _randn("fx", (1, 50, 3, 2, 32), (1, 50, 4), (32, 16))
        lens = torch.tensor([50], device=DEV)
        heads = lambda x, i: x[:, :, i].transpose(1, 2)  # noqa: E731
        f = ((lambda x: flash_spacetime_attention(heads(x, 0), heads(x, 1), heads(x, 2), feats, w, None, lens))
             if name == "attention" else lambda x: flash_spacetime_attention_qkv(x, feats, w, None, lens))
        tensors = [q]
    else:
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


def _block_run(blk, x, feats, dy, **kwargs):
    leaf = x.clone().requires_grad_(True)
    y = blk(leaf, feats, **kwargs)
    return y.detach(), torch.autograd.grad(y, [leaf, *blk.parameters()], dy.to(y.dtype))


@pytest.mark.parametrize("layout", ["lengths", "holes", "packed"])
@pytest.mark.parametrize("low", [torch.bfloat16, torch.float16], ids=["bf16", "f16"])
def test_block_under_autocast(low, layout):
    """float32 parameters and stream under autocast: output and gradients are float32
    and those of the float32 block up to the roundings of a 16-bit block (2e-2, the
    bound of the 16-bit attention module); so with the last sum deferred."""
    x, feats, dy = _randn(("autocast", layout), (3, 24, 64), (3, 24, 4), (3, 24, 64))
    blocks = [SpacetimeBlock(64, 4, device=DEV) for _ in range(2)]
    lens = torch.tensor([24, 7, 15], device=DEV)
    kwargs = {"seqlens": lens}
    if layout == "holes":
        kwargs = {"key_padding_mask": torch.arange(24, device=DEV)[None] % 5 >= 1 + torch.arange(3, device=DEV)[:, None]}
    elif layout == "packed":
        x, feats, dy = (t.flatten(0, 1) for t in (x, feats, dy))
        kwargs = {"cu_seqlens": torch.tensor([0, 30, 72], dtype=torch.int32, device=DEV)}
    near = lambda a, b: float((a - b).double().norm()) <= 2e-2 * float(b.double().norm())  # noqa: E731
    want = _block_run(blocks[0], x, feats, dy, **kwargs)
    with torch.autocast("cuda", dtype=low):
        got = _block_run(blocks[0], x, feats, dy, **kwargs)
        h, branch = blocks[0](x, feats, **kwargs, defer=True)
        two = blocks[1](h, feats, **kwargs, branch=branch).detach()
        again = blocks[1](got[0], feats, **kwargs).detach()
    assert branch.dtype == low and h.dtype == two.dtype == torch.float32
    assert got[0].dtype == torch.float32 and near(got[0], want[0]) and near(two, again)
    for a, b in zip(got[1], want[1]):
        assert a.dtype == torch.float32 and near(a, b)


def test_operators_under_autocast():
    """Tensors of one type keep their bits; of several they are what the casts
    written out give, gradients in the types that came in. Without autocast, and
    for float64, they are refused as before."""
    calls = _calls()
    for f, tensors in calls.values():
        want = f(*tensors)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            assert torch.equal(f(*tensors), want)
    low = torch.bfloat16
    f, (x, r, w) = calls["norm_residual"]
    g, ffn = calls["ffn"]
    with torch.autocast("cuda", dtype=low):
        for a, b, p in ((x.to(low), r, w), (x, r.to(low), w.to(low)), (x.half(), r.to(low), w.half()), (x, r, w.to(low)),
                        (x.half(), r.half(), w.to(low))):
            leaves = [t.detach().requires_grad_(True) for t in (a, b, p)]
            y = f(*leaves)
            wide = torch.promote_types(a.dtype, b.dtype)
            assert y.dtype == wide and torch.equal(y, f(a.to(wide), b.to(wide), p.float()))
            for t, d in zip(leaves, torch.autograd.grad(y, leaves, y.detach())):
                assert d.dtype == t.dtype and bool(d.isfinite().all()) and bool((d != 0).any())
        mixed = [ffn[0].half(), ffn[1], ffn[2].to(low), ffn[3]]
        leaves = [t.detach().requires_grad_(True) for t in mixed]
        y = g(*leaves)
        assert y.dtype == low and torch.equal(y, g(*(t.to(low) for t in mixed)))
        for t, d in zip(leaves, torch.autograd.grad(y, leaves, y.detach())):
            assert d.dtype == t.dtype and bool(d.isfinite().all()) and bool((d != 0).any())
        for bad in (lambda: f(x, r.double(), w), lambda: g(ffn[0].double(), *ffn[1:]), lambda: f(x[:1], r, w)):
            with pytest.raises(ValueError):
                bad()
    for bad in (lambda: f(x.to(low), r, w), lambda: g(ffn[0].to(low), *ffn[1:])):
        with pytest.raises(ValueError, match="dtype"):
            bad()
