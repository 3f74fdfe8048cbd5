"""GPU tests of packed events whose tensors are longer than their last offset (a
fixed number of tokens, as a captured graph has it): the tokens past it belong to
no event."""

import pytest
import torch

from tests._cases import seed_of

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from flash_spacetime_amd import SpacetimeAttention, _lib

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _leave_nan(*shapes):
    """Memory of these shapes, freed, that holds NaN: what rows left unwritten show."""
    for dtype in (torch.bfloat16, torch.float32):
        for _ in range(2):
            _ = [torch.full(s, float("nan"), device=DEV, dtype=dtype) for s in shapes for _ in range(4)]


@pytest.mark.parametrize("offsets,tokens,parts", [((0, 5, 9), 9, 3), ((0, 5, 9), 20, 3), ((0, 0), 7, 1), ((0,), 3, 2),
                                                  ((0, 900), 70001, 17), ((0, 30), 20, 2), ((0, 12, -4), 20, 2),
                                                  (tuple(range(700)), 800, 4)])
def test_zero_tail_writes_the_rows_past_every_offset(offsets, tokens, parts):
    cu = torch.tensor(offsets, dtype=torch.int32, device=DEV)
    rows = torch.ones(tokens + 2, 4 * parts, device=DEV)
    rc = _lib.load().fst_zero_tail(len(offsets) - 1, tokens, cu.data_ptr(), rows[1:].data_ptr(), 16 * parts,
                                   torch.cuda.current_stream().cuda_stream)
    assert rc == _lib.FST_OK
    want = torch.ones_like(rows)
    want[1 + min(max(offsets), tokens):1 + tokens] = 0
    assert torch.equal(rows, want)


def _grads(module, x, feats, cu, dy, **kwargs):
    x = x.clone().requires_grad_(True)
    y = module(x, feats, cu_seqlens=cu, **kwargs)
    _leave_nan(x.shape, (x.shape[0], 3 * x.shape[1]))
    return y.detach(), dict(zip(["x", *(n for n, _ in module.named_parameters())],
                       torch.autograd.grad(y, [x, *module.parameters()], dy)))


def _case(dtype, heads, key):
    gen = torch.Generator().manual_seed(seed_of("tail", dtype, key))
    dim, n, tokens = 16 * heads, 33, 47
    cu = torch.tensor([0, 20, 20, n], dtype=torch.int32, device=DEV)
    x = torch.randn(tokens, dim, generator=gen).to(DEV, TYPES[dtype])
    feats = torch.randn(tokens, 4, generator=gen).to(DEV)
    dy = torch.randn(tokens, dim, generator=gen).to(DEV, TYPES[dtype])
    dy[n:] = 0
    return dim, n, cu, x, feats, dy


@pytest.mark.parametrize("heads", [4, 20])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_attention_takes_nothing_in_from_tokens_of_no_event(dtype, heads):
    """SpacetimeAttention: the events' rows and every gradient are those of the call
    on the events' tokens alone. The linears' sums over tokens may be taken in
    another order: 2^-8 of a gradient's norm (float32 2^-20)."""
    dim, n, cu, x, feats, dy = _case(dtype, heads, heads)
    module = SpacetimeAttention(dim, heads, device=DEV, dtype=TYPES[dtype])
    _leave_nan((47, dim), (47, 3 * dim))
    y, got = _grads(module, x, feats, cu, dy)
    z, want = _grads(module, x[:n], feats[:n], cu, dy[:n])
    tol = 2.0 ** (-20 if dtype == "f32" else -8)
    assert float((y[:n] - z).double().norm()) <= tol * float(z.double().norm())
    assert bool(y.isfinite().all()) and bool((got["x"][n:] == 0).all())
    got["x"] = got["x"][:n]
    for name, w in want.items():
        assert float((got[name] - w).double().norm()) <= tol * float(w.double().norm()), name
