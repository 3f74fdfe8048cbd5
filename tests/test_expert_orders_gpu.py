"""The experts' movers on orders that were changed after the sort: slots taken out by their
places, experts cut off the table of offsets, rows that no slot has, in every width of a row's
group of lanes, on the host path and the Python path.

A slot has a row where 0 <= place < offsets[-1] and ys has that row. Bounds as
test_experts_gpu.py's: rows that are moved keep their bits, sums over K slots take K + 1
roundings of their terms, a dot at most 64.
"""

import pytest
import torch

from tests._block import TYPES
from tests._cases import seed_of
from tests._experts import sorted64

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from flash_spacetime_amd import (ExpertOrder, _lib, flash_expert_combine, flash_expert_dispatch, flash_expert_feed_forward,
                                     flash_expert_sort)

DEV = "cuda"
E = 2.0 ** -24


@pytest.fixture(params=["host", "python"])
def path(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(_lib, "_HOST", False)
    return request.param


def _gen(key):
    gen = torch.Generator().manual_seed(seed_of("orders", key))
    return gen, lambda *s: torch.randn(*s, generator=gen)


def _changed(tokens, k, n, drop, cut, gen):
    """A sorted order with some places taken out, and the last `cut` experts."""
    order = sorted64(torch.randint(0, n, (tokens, k), generator=gen), n)
    place = order[1].masked_fill(torch.rand(tokens, k, generator=gen) < drop, -1)
    return ExpertOrder(*(t.to(DEV) for t in (order[0], place, order[2][:n + 1 - cut])))


def _poison(*shapes, dtype):
    """Memory that the next allocations of these sizes find full of NaN."""
    for t in [torch.full(s, float("nan"), device=DEV, dtype=dtype) for s in shapes]:
        del t


def _run(x, ys, w, order, dxs, dy):
    x, ys, w = (t.detach().requires_grad_(True) for t in (x, ys, w))
    _poison(dxs.shape, ys.shape, x.shape, dtype=x.dtype)
    xs, y = flash_expert_dispatch(x, order), flash_expert_combine(ys, w, order)
    _poison(dxs.shape, ys.shape, x.shape, dtype=x.dtype)
    return [t.detach().double().cpu() for t in (xs, y, *torch.autograd.grad((xs, y), (x, ys, w), (dxs, dy)))]


def _check(x, ys, w, order, dxs, dy):
    xs, y, dx, dys, dw = _run(x, ys, w, order, dxs, dy)
    u = torch.finfo(x.dtype).eps / 2
    x, ys, w, dxs, dy = (t.detach().double().cpu() for t in (x, ys, w, dxs, dy))
    place, end = order.place.cpu().long(), int(order.offsets[-1])
    k = place.shape[1]

    def rows_of(t, slots):  # the slots' rows of t, zeros for those without
        has = (place >= 0) & (place < min(end, t.shape[0]))
        at = torch.where(has, place, t.shape[0])
        full = torch.cat([t, torch.zeros(1, t.shape[1], dtype=torch.float64)])
        return (full[at], has) if slots else has

    want, has = torch.zeros_like(xs), rows_of(dxs, False)
    want[place[has]] = x[:, None].expand(-1, k, -1)[has]
    assert torch.equal(xs, want), "xs"
    terms, has = rows_of(ys, True)
    terms = torch.where(has, w, 0.0)[..., None] * terms
    tiny = 2.0 ** -24
    assert bool(((y - terms.sum(1)).abs() <= u * terms.sum(1).abs() + (k + 1) * E * terms.abs().sum(1) + tiny).all()), "y"
    want = torch.zeros_like(dys)
    want[place[has]] = (w[..., None] * dy[:, None])[has]
    assert bool(((dys - want).abs() <= (u + 2 * E) * want.abs() + tiny).all()), "dys"
    terms = rows_of(ys, True)[0] * dy[:, None]
    assert bool(((dw - terms.sum(-1)).abs() <= 65 * E * terms.abs().sum(-1) + tiny).all()), "dweights"
    terms = rows_of(dxs, True)[0]
    assert bool(((dx - terms.sum(1)).abs() <= u * terms.sum(1).abs() + (k + 1) * E * terms.abs().sum(1) + tiny).all()), "dx"


def _case(dtype, tokens, k, d, rows, rn):
    t = TYPES[dtype]
    x, dy, ys, dxs = (rn(*s).to(DEV, t) for s in ((tokens, d), (tokens, d), (rows, d), (tokens * k, d)))
    return x, ys, rn(tokens, k).to(DEV), dxs, dy


@pytest.mark.parametrize("drop,cut", [(0.4, 0), (0.0, 3), (0.3, 2), (1.1, 0), (0.0, 7)])
@pytest.mark.parametrize("d", [1, 40, 384, 391, 1000, 2500, 8192])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_slots_taken_out_after_the_sort(path, dtype, d, drop, cut):
    gen, rn = _gen((dtype, d, drop, cut))
    tokens, k, n = 130, 3, 8
    order = _changed(tokens, k, n, drop, cut, gen)
    x, ys, w, dxs, dy = _case(dtype, tokens, k, d, tokens * k, rn)
    _check(x, ys, w, order, dxs, dy)


@pytest.mark.parametrize("rows", [0, 1, 150, 259, 261, 400])
def test_more_and_fewer_rows_than_slots(path, rows):
    """ys cut behind what it is needed for, or longer: places past its end add nothing, rows
    past the slots get a gradient of zeros."""
    gen, rn = _gen(("rows", rows))
    order = _changed(130, 2, 5, 0.2, 0, gen)
    x, ys, w, dxs, dy = _case("f32", 130, 2, 72, rows, rn)
    _check(x, ys, w, order, dxs, dy)


def test_many_rows_taken_out(path):
    gen, rn = _gen("many")
    order = _changed(60_000, 2, 16, 0.25, 1, gen)
    x, ys, w, dxs, dy = _case("bf16", 60_000, 2, 48, 120_000, rn)
    _check(x, ys, w, order, dxs, dy)


def test_a_capacity_reaches_the_experts_gradients(path):
    """Each expert keeps its first rows; what it loses is zeros between the runs, and the
    weights' gradients are those of the rows that are left."""
    gen, rn = _gen("capacity")
    tokens, k, n, d, f, cap = 200, 2, 4, 64, 96, 70
    order = flash_expert_sort(torch.randint(0, n, (tokens, k), generator=gen, dtype=torch.int32).to(DEV), n)
    first = order.offsets[:-1].long()
    of = torch.bucketize(order.place.long(), order.offsets[1:].long(), right=True)
    place = order.place.masked_fill(order.place - first[of] >= cap, -1)
    assert int((place < 0).sum()) > 0
    x, w = rn(tokens, d).to(DEV).requires_grad_(True), torch.rand(tokens, k, generator=gen).to(DEV)
    ws = [(0.1 * rn(*s)).to(DEV).requires_grad_(True) for s in ((n, f, d), (n, f, d), (n, d, f))]
    _poison((tokens * k, d), (tokens * k, d), dtype=torch.float32)
    kept = order._replace(place=place)
    y = flash_expert_combine(flash_expert_feed_forward(flash_expert_dispatch(x, kept), order.offsets, *ws), w, kept)
    _poison((tokens * k, d), (tokens * k, d), dtype=torch.float32)
    got = [y, *torch.autograd.grad(y, (x, *ws), torch.ones_like(y))]
    x64, ws64 = x.detach().double().requires_grad_(True), [v.detach().double().requires_grad_(True) for v in ws]
    y64 = 0.0
    for e in range(n):
        mine = (torch.where((of == e) & (place >= 0), w, 0.0)).double().sum(-1, keepdim=True)
        h = torch.nn.functional.silu(x64 @ ws64[0][e].t()) * (x64 @ ws64[1][e].t())
        y64 = y64 + mine * (h @ ws64[2][e].t())
    want = [y64, *torch.autograd.grad(y64, (x64, *ws64), torch.ones_like(y64))]
    for a, b in zip(got, want):
        assert float((a.double() - b).norm() / b.norm()) <= 1e-5


def test_places_change_between_replays():
    gen, rn = _gen("replays")
    order = _changed(300, 2, 6, 0.0, 0, gen)
    x, ys, w, dxs, dy = _case("f32", 300, 2, 96, 600, rn)
    place = order.place.clone()
    kept = order._replace(place=place)

    def step():
        leaves = [t.detach().requires_grad_(True) for t in (x, ys, w)]
        outs = flash_expert_dispatch(leaves[0], kept), flash_expert_combine(*leaves[1:], kept)
        return [*(o.detach() for o in outs), *torch.autograd.grad(outs, leaves, (dxs, dy))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
    for i in range(3):
        place.copy_(order.place.masked_fill(torch.rand(300, 2, generator=gen).to(DEV) < 0.3 * i, -1))
        want = step()
        torch.cuda.synchronize()
        for t in static:
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(static, want)), f"replay {i}"


def test_orders_are_checked(path):
    x, w = torch.randn(4, 16, device=DEV), torch.rand(4, 2, device=DEV)
    order = flash_expert_sort(torch.zeros(4, 2, dtype=torch.int32, device=DEV), 3)
    for bad in (order._replace(order=order.order.long()), order._replace(order=order.order.cpu()), order._replace(order=None)):
        with pytest.raises(ValueError, match="order.order"):
            flash_expert_dispatch(x, bad)
        with pytest.raises(ValueError, match="order.order"):
            flash_expert_combine(torch.randn(8, 16, device=DEV), w, bad)
