"""GPU parity of the mixture-of-experts operators against their definitions in 64 bits.

Bounds, derived before the first run. u is half a step of the output's type, e =
2^-24. Choices and orders are whole numbers and have to be equal. A weight is an
exponential of a difference l - top: the difference rounds once, which moves the
exponential by |l - top| e, its function by two units, sums of at most 512 terms (8 a
lane, then six levels), their quotient by one: (|l - top| + 24) e of its size. Rows that are
moved keep their bits; sums over a token's K slots take K + 1 roundings of the terms,
dots of D features at most 24 terms a lane, ten levels and the waves'. The
experts' feed-forward has flash_gated_feed_forward's bounds (test_feed_forward_gpu.py):
2 u of the 2-norm in 16-bit types, 5e-6 in float32, single rows four times as far.
"""

import pytest
import torch

from tests._block import TYPES, valid_rows
from tests._cases import seed_of
from tests._experts import expert_ffn64, route64, sorted64

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from flash_spacetime_amd import (ExpertOrder, flash_expert_combine, flash_expert_dispatch, flash_expert_feed_forward,
                                     flash_expert_route, flash_expert_sort)

DEV = "cuda"
E = 2.0 ** -24


def _u(dtype):
    return torch.finfo(dtype).eps / 2


def _gen(key):
    gen = torch.Generator().manual_seed(seed_of("experts", key))
    return lambda *s: torch.randn(*s, generator=gen)


def _within(name, got, want, bound):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, name
    far = (got - want).abs() - bound
    assert bool((far <= 0).all()), f"{name}: off by {(got - want).abs().max():.3e}, over its bound by {far.max():.3e}"


# --- router -----------------------------------------------------------------


def _check_route(logits, k, normalize, seqlens, dw):
    leaf = logits.detach().requires_grad_(True)
    weights, experts = flash_expert_route(leaf, k, normalize=normalize, seqlens=None if seqlens is None else seqlens.to(DEV))
    (grad,) = torch.autograd.grad(weights, leaf, dw)
    valid = valid_rows(logits.shape, seqlens)
    clean = torch.where(valid[..., None], logits.detach().cpu(), torch.zeros((), dtype=logits.dtype))
    w64, e64, g64 = route64(clean, k, normalize, valid, dw)
    assert experts.dtype == torch.int32 and weights.dtype == torch.float32 and grad.dtype == logits.dtype
    assert torch.equal(experts.cpu().long(), e64)
    v = clean.double()
    finite = torch.where(v == -torch.inf, 0.0, v)
    span = (finite.amax(-1, keepdim=True) - finite.amin(-1, keepdim=True)) + 24
    _within("weights", weights, w64, span * E * w64 + 2.0 ** -149)
    d = torch.where(valid[..., None], dw.double().cpu().abs(), 0.0)
    total = (w64 * d).sum(-1, keepdim=True)
    bound = torch.zeros_like(g64).scatter_add(-1, e64.clamp(min=0), w64 * (d + total))
    if not normalize:
        top = torch.where(e64[..., :1] >= 0, finite.amax(-1, keepdim=True), 0.0)
        p = torch.where(v == -torch.inf, 0.0, torch.exp(v - top))
        bound = bound + total * p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    tiny = torch.finfo(logits.dtype).smallest_normal * torch.finfo(logits.dtype).eps
    _within("dlogits", grad, g64, _u(logits.dtype) * g64.abs() + 4 * span * E * bound + tiny)
    with torch.no_grad():
        again = flash_expert_route(logits, k, normalize=normalize, seqlens=None if seqlens is None else seqlens.to(DEV))
        assert torch.equal(again[0], weights) and torch.equal(again[1], experts)


@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("n,k", [(1, 1), (2, 1), (2, 2), (5, 3), (8, 2), (16, 16), (17, 4), (64, 8), (65, 2), (127, 16), (128, 1),
                                 (129, 6), (300, 16), (512, 8)])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_routes(dtype, n, k, normalize):
    """16-bit logits of many experts hold many equal values: the lowest index wins."""
    rn = _gen((dtype, n, k))
    _check_route((2 * rn(173, n)).to(DEV, TYPES[dtype]), k, normalize, None, rn(173, k).to(DEV))


@pytest.mark.parametrize("normalize", [True, False])
def test_routes_of_padded_batches(normalize):
    rn = _gen(("padded", normalize))
    lens = torch.tensor([70, 0, 1, 129, 200, -2, 33])
    logits = rn(7, 129, 24)
    logits[~valid_rows(logits.shape, lens)] = float("nan")
    _check_route(logits.to(DEV), 3, normalize, lens, rn(7, 129, 3).to(DEV))


@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("n", [6, 40, 100, 400])
def test_masked_logits(n, normalize):
    """-inf is never chosen, also where it leaves fewer than top_k, or none; the type's lowest
    value and -0 are values like others."""
    rn = _gen(("masked", n, normalize))
    logits = rn(9, n)
    logits[0] = -torch.inf
    logits[1, :] = -torch.inf
    logits[1, n - 1] = 3.0
    logits[2, 1:] = -torch.inf
    logits[3] = torch.finfo(torch.float32).min
    logits[4] = 0.0
    logits[4, ::2] = -0.0
    logits[5, : n // 2] = -torch.inf
    _check_route(logits.to(DEV), 4, normalize, None, rn(9, 4).to(DEV))
    weights, experts = flash_expert_route(logits.to(DEV), 4, normalize=normalize)
    assert experts[0].tolist() == [-1] * 4 and experts[4].tolist() == [0, 1, 2, 3] and experts[1].tolist() == [n - 1, -1, -1, -1]
    assert bool((weights[0] == 0).all()) and float(weights[1, 0]) == 1.0


def test_logits_that_are_not_numbers():
    logits = torch.tensor([[1.0, float("nan"), 2.0, 0.5], [float("inf"), 0.0, 1.0, 2.0]], device=DEV)
    for normalize in (True, False):
        weights, experts = flash_expert_route(logits, 2, normalize=normalize)
        assert experts.tolist() == [[1, 2], [0, 3]] and bool(weights.isnan()[0].all()) and bool(weights.isnan()[1, 0])


def test_route_strides_and_rows():
    rn = _gen("route strides")
    wide = rn(30, 100).to(DEV)
    want = flash_expert_route(wide[:, 7:40].contiguous(), 3)
    for view in (wide[:, 7:40], wide[:, 7:40].t().contiguous().t()):
        assert all(torch.equal(a, b) for a, b in zip(flash_expert_route(view, 3), want))
    for rows in (0, 1, 15, 16, 17):
        got = flash_expert_route(wide[:rows, 7:40], 3)
        assert all(torch.equal(a, b[:rows]) for a, b in zip(got, want))
    leaf = wide[:0].clone().requires_grad_(True)
    assert torch.autograd.grad(flash_expert_route(leaf, 2)[0].sum(), leaf)[0].shape == (0, 100)


# --- sort -------------------------------------------------------------------


@pytest.mark.parametrize("slots,k,n", [(0, 1, 3), (1, 1, 1), (2, 2, 5), (63, 1, 4), (64, 2, 8), (1000, 4, 64), (8192, 2, 16),
                                       (8196, 4, 16), (40000, 8, 512), (200001, 3, 65), (786432, 4, 64), (50000, 1, 1),
                                       (30000, 2, 300)])
@pytest.mark.parametrize("kind", ["all", "some", "skewed"])
def test_sorts(slots, k, n, kind):
    gen = torch.Generator().manual_seed(seed_of("sort", slots, k, n, kind))
    lo, hi = (0, n) if kind == "all" else (-2, n + 2)
    experts = torch.randint(lo, hi, (slots // k, k), generator=gen, dtype=torch.int32)
    if kind == "skewed":
        experts[torch.rand(experts.shape, generator=gen) < 0.8] = n // 2
    got = flash_expert_sort(experts.to(DEV), n)
    assert isinstance(got, ExpertOrder)
    for name, a, b in zip(got._fields, got, sorted64(experts, n)):
        assert a.dtype == torch.int32 and torch.equal(a.cpu(), b), name


def test_sorts_as_many_slots_as_there_may_be():
    """2^31 - 65537 of them, expert by expert in turn: each one's row and slot by arithmetic."""
    n, e, chunk = 0x7FFFFFFF - 65536, 5, 1 << 28
    spans = [(a, min(n, a + chunk)) for a in range(0, n, chunk)]
    ids = torch.empty(n, 1, dtype=torch.int32, device=DEV)
    for a, b in spans:
        ids[a:b, 0] = torch.arange(a, b, device=DEV) % (e + 1)  # the last: no expert
    got = flash_expert_sort(ids, e)
    del ids
    counts = [(n + e - i) // (e + 1) for i in range(e)]
    assert got.offsets.tolist() == [sum(counts[:i]) for i in range(e + 1)]
    offsets = got.offsets.long()
    for a, b in spans:
        slot = torch.arange(a, b, device=DEV)
        of = slot % (e + 1)
        assert torch.equal(got.place[a:b, 0], torch.where(of == e, -1, offsets[of] + slot // (e + 1)).int())
        of = torch.bucketize(slot, offsets[1:], right=True)
        want = torch.where(of == e, -1, (slot - offsets[of]) * (e + 1) + of)
        assert torch.equal(got.order[a:b], want.int())


def test_sorts_other_integers_and_strides():
    experts = torch.tensor([[3, 1 << 32, -7], [0, 3, (1 << 40) + 1]])
    want = sorted64(torch.tensor([[3, -1, -1], [0, 3, -1]]), 4)
    for t in (experts.to(DEV), experts.to(DEV).t().contiguous().t()):
        assert all(torch.equal(a.cpu(), b) for a, b in zip(flash_expert_sort(t, 4), want))
    small = torch.tensor([[2, 0], [1, 2]], dtype=torch.uint8)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(flash_expert_sort(small.to(DEV), 3), sorted64(small, 3)))


# --- rows to the experts and back -------------------------------------------


def _order(tokens, k, n, drop, key):
    gen = torch.Generator().manual_seed(seed_of("order", key))
    experts = torch.stack([torch.randperm(max(n, k), generator=gen)[:k] for _ in range(tokens)]) if tokens else torch.zeros(0, k)
    experts = experts.int()
    if drop:
        experts[torch.rand(experts.shape, generator=gen) < drop] = -1
    return ExpertOrder(*(t.to(DEV) for t in sorted64(experts, n)))


def _check_shuffle(x, ys, w, order, dxs, dy, got):
    xs, y, dx, dys, dw = got
    place = order.place.cpu().long()
    lead, k, d, rows = place.shape[:-1], place.shape[-1], x.shape[-1], ys.shape[0]
    at = torch.where(place < 0, rows, place).reshape(-1)

    def spread(t):
        full = torch.zeros(rows + 1, d, dtype=torch.float64)
        full[at] = t.reshape(-1, d)
        return full[:rows]

    def back(t):
        return torch.cat([t.detach().double().cpu(), torch.zeros(1, d, dtype=torch.float64)])[at].reshape(*lead, k, d)

    c = lambda t: t.detach().double().cpu()  # noqa: E731
    u, tiny = _u(x.dtype), torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    assert torch.equal(c(xs), spread(c(x)[..., None, :].expand(*lead, k, d))), "xs"
    w64 = torch.where(place < 0, 0.0, c(w))[..., None]
    terms = w64 * back(ys)
    _within("y", y, terms.sum(-2), u * terms.sum(-2).abs() + (k + 1) * E * terms.abs().sum(-2) + tiny)
    terms = back(dxs)
    _within("dx", dx, terms.sum(-2), u * terms.sum(-2).abs() + (k + 1) * E * terms.abs().sum(-2) + tiny)
    want = spread(w64 * c(dy)[..., None, :])
    _within("dys", dys, want, (u + 2 * E) * want.abs() + tiny)
    terms = c(dy)[..., None, :] * back(ys)
    _within("dweights", dw, terms.sum(-1), _u(w.dtype) * terms.sum(-1).abs() + 64 * E * terms.abs().sum(-1) + tiny)


def _shuffle(x, ys, w, order, dxs, dy):
    x, ys, w = (t.detach().requires_grad_(True) for t in (x, ys, w))
    xs, y = flash_expert_dispatch(x, order), flash_expert_combine(ys, w, order)
    return [xs, y, *torch.autograd.grad((xs, y), (x, ys, w), (dxs, dy))]


@pytest.mark.parametrize("tokens,k,n,drop", [(0, 2, 4, 0), (1, 1, 1, 0), (3, 2, 4, 0.5), (187, 2, 8, 0), (200, 1, 16, 0.9),
                                             (333, 16, 20, 0.3), (50, 4, 8, 1.1)])
@pytest.mark.parametrize("d", [1, 3, 8, 71, 384, 1000, 4096, 8192])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_rows_to_the_experts_and_back(dtype, d, tokens, k, n, drop):
    t = TYPES[dtype]
    rn = _gen((dtype, d, tokens, k))
    order = _order(tokens, k, n, drop, (tokens, k, n))
    rows = tokens * k
    w = torch.softmax(rn(tokens, k), -1).to(DEV, torch.float32 if d % 2 else t)
    x, ys, dxs, dy = (rn(*s).to(DEV, t) for s in ((tokens, d), (rows, d), (rows, d), (tokens, d)))
    got = _shuffle(x, ys, w, order, dxs, dy)
    _check_shuffle(x, ys, w, order, dxs, dy, got)


def test_rows_of_many_tokens():
    """More rows than a grid's groups take at once, in a padded batch."""
    rn = _gen("many")
    b, length, k, n, d = 40, 2000, 2, 8, 96
    lens = torch.randint(0, length + 1, (b,), generator=torch.Generator().manual_seed(3))
    experts = torch.randint(0, n, (b, length, k), generator=torch.Generator().manual_seed(4), dtype=torch.int32)
    experts[~valid_rows((b, length, k), lens)] = -1
    order = flash_expert_sort(experts.to(DEV), n)
    rows = b * length * k
    x, dy = rn(b, length, d).to(DEV, torch.bfloat16), rn(b, length, d).to(DEV, torch.bfloat16)
    ys, dxs = rn(rows, d).to(DEV, torch.bfloat16), rn(rows, d).to(DEV, torch.bfloat16)
    # What has no place holds anything, and is not read.
    pad = ~valid_rows(x.shape, lens).to(DEV)
    x[pad] = float("nan")
    used = int(order.offsets[-1])
    ys[used:], dxs[used:] = float("inf"), float("nan")
    w = rn(b, length, k).to(DEV)
    w[pad] = float("nan")
    got = _shuffle(x, ys, w, order, dxs, dy)
    assert bool((got[0][used:] == 0).all()) and bool((got[1].detach()[pad] == 0).all())
    clean = lambda t, m: torch.where(m, 0.0, t).to(t.dtype)  # noqa: E731
    tail = (torch.arange(rows, device=DEV) >= used)[:, None]
    _check_shuffle(clean(x, pad[..., None]), clean(ys, tail), clean(w, pad[..., None]), order, clean(dxs, tail), dy, got)


def test_shuffle_strides_and_single_gradients():
    rn = _gen("shuffle strides")
    order = _order(60, 2, 6, 0.2, "strides")
    x, dy = rn(60, 128).to(DEV), rn(60, 128).to(DEV)
    ys, dxs, w = rn(120, 128).to(DEV), rn(120, 128).to(DEV), torch.rand(60, 2).to(DEV)
    want = _shuffle(x, ys, w, order, dxs, dy)
    off = lambda t: torch.cat([t.new_zeros(t.shape[0], 3), t], 1)[:, 3:]  # noqa: E731
    turned = lambda t: t.t().contiguous().t()  # noqa: E731
    for f in (off, turned):
        got = _shuffle(f(x), f(ys), turned(w), order, f(dxs), f(dy))
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    one = dy[:1].expand(60, 128)
    a, b = _shuffle(x, ys, w, order, dxs, one), _shuffle(x, ys, w, order, dxs, one.contiguous())
    assert all(torch.equal(i, j) for i, j in zip(a, b))
    for i in range(2):
        leaves = [ys.detach().requires_grad_(i == 0), w.detach().requires_grad_(i == 1)]
        (grad,) = torch.autograd.grad(flash_expert_combine(*leaves, order), leaves[i], dy)
        assert torch.equal(grad, want[3 + i])


# --- the experts' feed-forward ----------------------------------------------

NAMES = ("y", "dx", "dw_gate", "dw_up", "dw_down")


def _near(name, got, want, tol):
    got, want = got.detach().double(), want.to(got.device)
    assert got.shape == want.shape, name
    err = float((got - want).norm() / want.norm().clamp_min(1e-30))
    assert err <= tol, f"{name}: relative error {err:.3e} over {tol:.1e}"
    if got.numel():
        rows, ref = (got - want).flatten(0, -2).norm(dim=-1), want.flatten(0, -2).norm(dim=-1)
        typical = ref.square().mean().sqrt()
        far = float((rows / (ref + 0.1 * typical).clamp_min(1e-30)).max())
        assert far <= 4 * tol, f"{name}: a row's relative error {far:.3e}"


def _tol(dtype):
    return 5e-6 if dtype == torch.float32 else torch.finfo(dtype).eps


def _ffn_case(loads, d, f, dtype, key, tail=0):
    rn = _gen(("ffn", key))
    n, rows = len(loads), sum(loads) + tail
    x, dy = rn(rows, d).to(DEV, dtype), rn(rows, d).to(DEV, dtype)
    ws = [(rn(n, f, d) / d ** 0.5).to(DEV, dtype), (rn(n, f, d) / d ** 0.5).to(DEV, dtype), (rn(n, d, f) / f ** 0.5).to(DEV, dtype)]
    offsets = torch.tensor([0, *loads]).cumsum(0).int().to(DEV)
    return x, ws, offsets, dy


def _ffn(x, offsets, ws, act, dy):
    leaves = [t.detach().requires_grad_(True) for t in (x, *ws)]
    y = flash_expert_feed_forward(leaves[0], offsets, *leaves[1:], act)
    return [y, *torch.autograd.grad(y, leaves, dy)]


def _check_ffn(x, ws, offsets, dy, act):
    got = _ffn(x, offsets, ws, act, dy)
    used = int(offsets[-1])
    assert all(bool((t.detach()[used:] == 0).all()) for t in got[:2])
    want = expert_ffn64(x[:used], offsets, *ws, act, dy[:used])
    for name, a, b in zip(NAMES, got, want):
        _near(name, a[:used] if name in ("y", "dx") else a, b, _tol(x.dtype))
    for e in range(len(offsets) - 1):
        if int(offsets[e]) == int(offsets[e + 1]):
            assert all(bool((t[e] == 0).all()) for t in got[2:]), "gradients of an expert without rows"
    with torch.no_grad():
        assert torch.equal(flash_expert_feed_forward(x, offsets, *ws, act), got[0])


LOADS = [
    ([1], 8, 8), ([0], 64, 64), ([0, 3, 0, 5], 16, 24), ([17], 32, 64), ([8] * 8, 768, 264), ([64], 64, 128), ([20, 0, 33], 40, 72),
    ([1] * 65, 64, 64), ([100, 1, 0, 86], 384, 512), ([63, 64, 65, 66], 136, 520), ([0, 0, 513], 96, 1000), ([500, 200, 300], 384, 256),
    ([3] * 200, 72, 136), ([2050, 0, 1, 77, 900], 256, 320), ([257, 255, 256, 1], 384, 640), ([1000] * 8, 128, 200),
]


@pytest.mark.parametrize("loads,d,f", LOADS, ids=[f"{len(x[0])}x{sum(x[0])}_{x[1]}_{x[2]}" for x in LOADS])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_expert_feed_forward(dtype, loads, d, f):
    act = ("silu", "gelu", "gelu_tanh")[(len(loads) + f // 8) % 3]
    x, ws, offsets, dy = _ffn_case(loads, d, f, TYPES[dtype], (dtype, tuple(loads), d, f))
    _check_ffn(x, ws, offsets, dy, act)


@pytest.mark.parametrize("loads,tail", [([5, 0, 7], 20), ([0, 0], 90), ([300, 10, 0, 200], 1), ([700, 900], 2000), ([3000] * 6, 18000)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_rows_past_the_last_expert(dtype, loads, tail):
    """They hold anything and reach nothing."""
    x, ws, offsets, dy = _ffn_case(loads, 192, 256, TYPES[dtype], (dtype, tuple(loads), "tail"), tail)
    used = sum(loads)
    x[used:], dy[used:] = float("nan"), float("inf")
    _check_ffn(x, ws, offsets, dy, "silu")


@pytest.mark.parametrize("loads", [[3, 5, 0, 7], [40, 100, 0, 60, 33], [700, 300, 900, 400]])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_a_part_of_the_experts(dtype, loads):
    """Offsets cut out of a longer table: rows before and behind are zeros, and what they
    hold reaches nothing; the others have the whole call's bits."""
    x, ws, offsets, dy = _ffn_case(loads, 64, 128, TYPES[dtype], (dtype, tuple(loads), "part"), tail=50)
    want = _ffn(x, offsets, ws, "silu", dy)
    lo, hi = int(offsets[1]), int(offsets[3])
    x, dy = x.clone(), dy.clone()
    for t, what in ((x, float("nan")), (dy, float("inf"))):
        t[:lo], t[hi:] = what, what
    got = _ffn(x, offsets[1:4], [w[1:3] for w in ws], "silu", dy)
    for a, b in zip(got[:2], want[:2]):
        assert bool((a[:lo] == 0).all()) and bool((a[hi:] == 0).all()) and torch.equal(a[lo:hi], b[lo:hi])
    used = expert_ffn64(x[lo:hi], offsets[1:4] - offsets[1], *(w[1:3] for w in ws), "silu", dy[lo:hi])
    for name, a, b in zip(NAMES[2:], got[2:], used[2:]):
        _near(name, a, b, _tol(TYPES[dtype]))


def test_no_rows():
    x, ws, offsets, dy = _ffn_case([0, 0, 0], 64, 128, torch.bfloat16, "none")
    got = _ffn(x, offsets, ws, "silu", dy)
    assert got[0].shape == got[1].shape == (0, 64) and all(bool((t == 0).all()) for t in got[2:])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_feed_forward_strides_and_single_gradients(dtype):
    x, ws, offsets, dy = _ffn_case([40, 0, 160], 64, 96, TYPES[dtype], "strides")
    want = _ffn(x, offsets, ws, "gelu", dy)
    wide = torch.zeros(200, 128, device=DEV, dtype=x.dtype)
    wide[:, 32:96] = x
    off = torch.zeros(200, 67, device=DEV, dtype=x.dtype)[:, 3:]
    off.copy_(dy)
    turned = [w.transpose(1, 2).contiguous().transpose(1, 2) for w in ws]
    got = _ffn(wide[:, 32:96], offsets, turned, "gelu", off)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for i in range(4):
        leaves = [t.detach().requires_grad_(i == j) for j, t in enumerate((x, *ws))]
        y = flash_expert_feed_forward(leaves[0], offsets, *leaves[1:], "gelu")
        assert torch.equal(torch.autograd.grad(y, leaves[i], dy)[0], want[1 + i]), NAMES[1 + i]


# --- together ---------------------------------------------------------------


def _mixture(x, logits, ws, k, lens):
    weights, experts = flash_expert_route(logits, k, seqlens=lens)
    order = flash_expert_sort(experts, logits.shape[-1])
    rows = flash_expert_feed_forward(flash_expert_dispatch(x, order), order.offsets, *ws)
    return flash_expert_combine(rows, weights, order)


def _mixture64(x, logits, ws, k, valid):
    """The mixture by its definition, every expert on every token, in float64 with a graph."""
    v = torch.sort(-logits.detach(), dim=-1, stable=True).indices[..., :k]
    w = torch.softmax(torch.gather(logits, -1, v), -1)
    y = 0.0
    for e in range(logits.shape[-1]):
        h = torch.nn.functional.silu(x @ ws[0][e].t()) * (x @ ws[1][e].t())
        y = y + (w * (v == e)).sum(-1, keepdim=True) * (h @ ws[2][e].t())
    return torch.where(valid[..., None], y, 0.0)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_a_mixture_of_experts(dtype):
    """The operators in a row, forward and backward. 16-bit rows take three more roundings
    than the feed-forward alone (its rows, and the gradients of both movers): 4 u of the
    norm is allowed, 1e-5 in float32."""
    t, (b, length, d, f, n, k) = TYPES[dtype], (5, 70, 128, 192, 9, 3)
    rn = _gen(("mixture", dtype))
    lens = torch.tensor([70, 3, 0, 51, 66])
    valid = valid_rows((b, length, d), lens)
    x, logits, dy = rn(b, length, d).to(t), rn(b, length, n), rn(b, length, d).to(t)
    ws = [(rn(n, f, d) / d ** 0.5).to(t), (rn(n, f, d) / d ** 0.5).to(t), (rn(n, d, f) / f ** 0.5).to(t)]
    leaves = [v.to(DEV).requires_grad_(True) for v in (x, logits, *ws)]
    y = _mixture(leaves[0], leaves[1], leaves[2:], k, lens.to(DEV))
    got = [y, *torch.autograd.grad(y, leaves, dy.to(DEV))]
    exact = [v.double().requires_grad_(True) for v in (x, logits, *ws)]
    y64 = _mixture64(exact[0], exact[1], exact[2:], k, valid)
    want = [y64.detach(), *torch.autograd.grad(y64, exact, dy.double())]
    for name, a, c in zip(("y", "dx", "dlogits", "dw_gate", "dw_up", "dw_down"), got, want):
        _near(name, a, c, 1e-5 if dtype == "f32" else 4 * _u(t))


def test_a_mixture_replays_in_a_graph():
    """Loads that change between replays; two graphs share nothing."""
    rn = _gen("graph")
    d, f, n, k = 128, 192, 8, 2
    x, dy = rn(6, 90, d).to(DEV, torch.bfloat16), rn(6, 90, d).to(DEV, torch.bfloat16)
    logits = rn(6, 90, n).to(DEV)
    ws = [(rn(*s) / 12).to(DEV, torch.bfloat16) for s in ((n, f, d), (n, f, d), (n, d, f))]
    lens = torch.tensor([90, 3, 0, 17, 88, 1], device=DEV, dtype=torch.int32)

    def step():
        leaves = [t.detach().requires_grad_(True) for t in (x, logits, *ws)]
        y = _mixture(leaves[0], leaves[1], leaves[2:], k, lens)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, step()))
    for i in range(3):
        logits.copy_(torch.randn_like(logits) * (1 + 4 * i))
        lens.copy_(torch.roll(lens, 1))
        want = step()
        torch.cuda.synchronize()
        for graph, static in graphs:
            for t in static:
                t.fill_(float("nan"))
        for graph, static in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, static in graphs:
            assert all(torch.equal(a, c) for a, c in zip(static, want)), f"replay {i}"


def test_results_repeat_bitwise():
    rn = _gen("repeat")
    x, logits = rn(3000, 128).to(DEV, torch.bfloat16), rn(3000, 16).to(DEV)
    ws = [(rn(*s) / 12).to(DEV, torch.bfloat16) for s in ((16, 192, 128), (16, 192, 128), (16, 128, 192))]

    def step():
        leaves = [t.detach().requires_grad_(True) for t in (x, logits, *ws)]
        y = _mixture(leaves[0], leaves[1], leaves[2:], 2, None)
        return [y.detach(), *torch.autograd.grad(y.float().square().sum(), leaves)]

    want = step()
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(step(), want))


# --- sizes past 32 bits, and nothing at all -----------------------------------


def test_rows_past_32_bits():
    """280000 rows of 8192: byte and element offsets of the last rows pass 2^32 and 2^31."""
    tokens, d, n = 280_000, 8192, 3
    experts = torch.randint(0, n, (tokens, 1), generator=torch.Generator().manual_seed(1), dtype=torch.int32)
    order = flash_expert_sort(experts.to(DEV), n)
    x = torch.empty(tokens, d, device=DEV, dtype=torch.bfloat16)
    x.copy_((torch.arange(tokens, device=DEV) % 251)[:, None] + (torch.arange(d, device=DEV) % 4)[None, :])
    w = torch.full((tokens, 1), 0.5, device=DEV)
    leaves = [x.requires_grad_(True), w.requires_grad_(True)]
    xs = flash_expert_dispatch(leaves[0], order)
    y = flash_expert_combine(xs, leaves[1], order)
    dx, dw = torch.autograd.grad(y, leaves, x.detach())
    at = torch.tensor([0, 1, 131_071, 140_001, 262_143, 262_145, tokens - 1])
    place = order.place[:, 0].long()[at]
    assert torch.equal(xs.detach()[place], x.detach()[at])
    assert torch.equal(y.detach()[at], 0.5 * x.detach()[at]) and torch.equal(dx[at], 0.5 * x.detach()[at])
    want = x.detach()[at].double().square().sum(-1)
    assert bool(((dw[at, 0].double() - want).abs() <= 64 * E * want).all())


def test_feed_forward_past_32_bits():
    """The gradients' rows of 2 F: 300000 x 8192. Rows near either end against 64 bits."""
    loads, d, f = [150_000, 0, 150_000], 64, 4096
    x, ws, offsets, dy = _ffn_case([5], d, f, torch.bfloat16, "wide")
    rn = _gen("past 32 bits")
    x, dy = (rn(sum(loads), d).to(DEV, torch.bfloat16) for _ in range(2))
    ws = [(rn(3, *w.shape[1:]) / w.shape[2] ** 0.5).to(DEV, torch.bfloat16) for w in ws]
    offsets = torch.tensor([0, *loads]).cumsum(0).int().to(DEV)
    got = _ffn(x, offsets, ws, "silu", dy)
    for lo, hi, e in ((0, 500, 0), (149_500, 150_000, 0), (299_500, 300_000, 2)):
        one = expert_ffn64(x[lo:hi], torch.tensor([0, hi - lo]), *(w[e:e + 1] for w in ws), "silu", dy[lo:hi])
        _near("y", got[0][lo:hi], one[0], _tol(torch.bfloat16))
        _near("dx", got[1][lo:hi], one[1], _tol(torch.bfloat16))
    # dw_down of an expert, formed by halves of its rows
    half = [expert_ffn64(x[lo:lo + 75_000], torch.tensor([0, 75_000]), *(w[2:] for w in ws), "silu", dy[lo:lo + 75_000])
            for lo in (150_000, 225_000)]
    for i, name in enumerate(NAMES[2:]):
        _near(name, got[2 + i][2], (half[0][2 + i] + half[1][2 + i])[0], _tol(torch.bfloat16))
        assert bool((got[2 + i][1] == 0).all())


def test_tokens_without_rows_and_rows_without_tokens():
    none = torch.full((5, 2), -1, dtype=torch.int32, device=DEV)
    order = ExpertOrder(none[:, 0], none, torch.zeros(4, dtype=torch.int32, device=DEV))
    ys = torch.empty(0, 48, device=DEV, requires_grad=True)
    w = torch.full((5, 2), float("nan"), device=DEV, requires_grad=True)
    y = flash_expert_combine(ys, w, order)
    assert bool((y == 0).all())
    dys, dw = torch.autograd.grad(y, (ys, w), torch.ones_like(y))
    assert dys.shape == (0, 48) and bool((dw == 0).all())
    order = flash_expert_sort(torch.empty(0, 2, dtype=torch.int32, device=DEV), 3)
    ys = torch.full((7, 48), float("nan"), device=DEV, requires_grad=True)
    w = torch.empty(0, 2, device=DEV, requires_grad=True)
    y = flash_expert_combine(ys, w, order)
    dys, dw = torch.autograd.grad(y, (ys, w), torch.ones_like(y))
    assert y.shape == (0, 48) and dw.shape == (0, 2) and bool((dys == 0).all())
    assert flash_expert_dispatch(torch.empty(0, 48, device=DEV), order).shape == (0, 48)


@pytest.mark.parametrize("n", [1, 64, 65, 130, 300, 512])
def test_as_many_experts_as_there_may_be(n):
    """Runs are looked up 64 experts at a time; some are empty, the last ones not."""
    loads = [(e * 7) % 5 * (e % 3 != 0) for e in range(n)]
    loads[-1] = 3
    x, ws, offsets, dy = _ffn_case(loads, 32, 40, torch.bfloat16, ("many experts", n), tail=6)
    _check_ffn(x, ws, offsets, dy, "silu")
