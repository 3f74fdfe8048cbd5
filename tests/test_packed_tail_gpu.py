"""GPU tests of packed events whose tensors are longer than their last offset (a
fixed number of tokens, as a captured graph has it): the tokens past it belong to
no event."""

import pytest
import torch

from tests._cases import seed_of

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from flash_spacetime_amd import (SpacetimeAttention, SpacetimeBlock, _lib, flash_gated_feed_forward,
                                     flash_layer_norm)

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


@pytest.mark.parametrize("branch", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_block_leaves_tokens_of_no_event_alone(dtype, branch):
    """SpacetimeBlock: what those tokens hold (NaN and infinities) and what their
    gradient is changes nothing; output and x's gradient there are zeros."""
    dim, n, cu, x, feats, dy = _case(dtype, 4, branch)
    module = SpacetimeBlock(dim, 4, device=DEV, dtype=TYPES[dtype])
    x[n:], feats[n:], dy[n:] = float("nan"), float("inf"), float("nan")
    kw = {"branch": x.flip(1)} if branch else {}
    kw_n = {k: v[:n] for k, v in kw.items()}
    _leave_nan((47, dim), (47, 3 * dim), (47, 192))
    y, got = _grads(module, x, feats, cu, dy, **kw)
    z, want = _grads(module, x[:n], feats[:n], cu, dy[:n], **kw_n)
    assert bool((y[n:] == 0).all()) and bool((got["x"][n:] == 0).all())
    tol = 2.0 ** (-20 if dtype == "f32" else -8)
    assert float((y[:n] - z).double().norm()) <= tol * float(z.double().norm())
    got["x"] = got["x"][:n]
    for name, w in want.items():
        assert float((got[name] - w).double().norm()) <= tol * float(w.double().norm()), name


def test_block_in_a_graph_whose_offsets_change():
    """A captured forward and backward of a fixed number of tokens, replayed for
    other events: each replay has the eager call's bits."""
    dim, n, cu, x, feats, dy = _case("bf16", 4, "graph")
    dy = x.flip(0).contiguous()
    module = SpacetimeBlock(dim, 4, device=DEV, dtype=torch.bfloat16)

    def step():
        leaves = [x.detach().requires_grad_(True), *module.parameters()]
        y = module(leaves[0], feats, cu_seqlens=cu)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
    for offsets in ((0, 20, 20, 33), (0, 1, 40, 47), (0, 0, 0, 0), (0, 17, 30, 31)):
        cu.copy_(torch.tensor(offsets, dtype=torch.int32))
        for t in static:
            t.fill_(float("nan"))
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(static, want):
            assert torch.equal(a, b), offsets


def test_block_refuses_offsets_of_another_shape():
    module = SpacetimeBlock(64, 4, device=DEV)
    x, feats = torch.randn(9, 64, device=DEV), torch.randn(9, 4, device=DEV)
    for cu in (torch.zeros(0, dtype=torch.int32, device=DEV), torch.zeros(1, 2, dtype=torch.int32, device=DEV)):
        with pytest.raises(ValueError, match="cu_seqlens"):
            module(x, feats, cu_seqlens=cu)


@pytest.mark.parametrize("tokens", [-1, 0, 1, 20, 29, 40])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_operators_take_packed_rows_with_one_length(monkeypatch, dtype, tokens):
    """x [T, N] with seqlens [1]: the bits of the padded batch of one event, through the
    host extension and without it."""
    gen = torch.Generator().manual_seed(5)
    rn = lambda *s: torch.randn(*s, generator=gen).to(DEV, TYPES[dtype])  # noqa: E731
    x, r, w, dy = rn(29, 64), rn(29, 64), rn(64), rn(29, 64)
    ws = [rn(128, 64) / 8, rn(128, 64) / 8, rn(64, 128) / 11]
    lens = torch.tensor([tokens], device=DEV)

    def run(see, back):
        leaves = [t.detach().requires_grad_(True) for t in (x, r, w, *ws)]
        a, b = see(leaves[0]), see(leaves[1])
        y, s = flash_layer_norm(a, leaves[2], residual=b, seqlens=lens)
        z = flash_gated_feed_forward(y, *leaves[3:], seqlens=lens)
        return [back(y), back(z), *torch.autograd.grad((z, s), leaves, (see(dy), see(dy)))]

    want = run(lambda t: t[None], lambda t: t[0])
    assert bool((want[1][max(tokens, 0):] == 0).all())
    for host in (True, False):
        with monkeypatch.context() as m:
            if not host:
                m.setattr(_lib, "host", lambda: None)
            got = run(lambda t: t, lambda t: t)
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    for bad in (torch.tensor([3, 4], device=DEV), torch.tensor([[3]], device=DEV)):
        with pytest.raises(ValueError, match="padded"):
            flash_layer_norm(x, seqlens=bad)
        with pytest.raises(ValueError, match="padded"):
            flash_gated_feed_forward(x, *ws, seqlens=bad)


@pytest.mark.parametrize("kind", ["int64", "host", "strided"])
def test_block_takes_offsets_of_any_kind(kind):
    dim, n, cu, x, feats, dy = _case("f32", 4, "kinds")
    module = SpacetimeBlock(dim, 4, device=DEV)
    other = {"int64": cu.long(), "host": cu.cpu(), "strided": torch.stack([cu, cu + 99], 1)[:, 0]}[kind]
    y, want = _grads(module, x, feats, cu, dy)
    z, got = _grads(module, x, feats, other, dy)
    assert torch.equal(y, z) and bool((y[n:] == 0).all())
    for name, w in want.items():
        assert torch.equal(got[name], w), name
