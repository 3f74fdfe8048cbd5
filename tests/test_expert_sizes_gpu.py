"""The experts' operators at sizes past those that one launch, or 32 bits, take."""

import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from flash_spacetime_amd import flash_expert_feed_forward, flash_expert_route, flash_gated_feed_forward

DEV = "cuda"


@pytest.mark.parametrize("rows,n,k", [((1 << 26) + 777, 129, 1), ((1 << 28) + 4099, 65, 1), ((1 << 29) + 515, 2, 1)])
def test_routes_of_more_rows_than_a_launch_takes(rows, n, k):
    """64, 16 and 8 lanes a row: 2^32 lanes at 2^26, 2^28 and 2^29 rows. Every row holds the
    logits of one of 61, so that what it has to give is the small call's."""
    kinds = torch.randn(61, n, generator=torch.Generator().manual_seed(n)).to(DEV, torch.bfloat16)
    logits = torch.empty(rows, n, device=DEV, dtype=torch.bfloat16)
    chunk = 61 << 16
    of = torch.arange(chunk, device=DEV) % 61
    for a in range(0, rows, chunk):  # chunk is a multiple of 61
        logits[a:a + chunk] = kinds[of[: rows - a]]
    leaf = logits.requires_grad_(True)
    weights, experts = flash_expert_route(leaf, k)
    small = kinds.requires_grad_(True)
    want_w, want_e = flash_expert_route(small, k)
    dw = torch.arange(1, k + 1, device=DEV, dtype=torch.float32)
    (want_g,) = torch.autograd.grad(want_w, small, dw.expand(61, k))
    for a in range(0, rows, chunk):
        here = of[: rows - a]
        assert torch.equal(weights[a:a + chunk], want_w[here]) and torch.equal(experts[a:a + chunk], want_e[here])
    (grad,) = torch.autograd.grad(weights, leaf, dw.expand(rows, k))
    for a in range(0, rows, chunk):
        assert torch.equal(grad[a:a + chunk], want_g[of[: rows - a]])


@pytest.mark.parametrize("experts", [None, 3])
def test_feed_forward_of_more_rows_than_a_launch_takes(experts):
    """2^30 rows of 8 features: the output product's tiles of 64 rows, and the backward's,
    have 2^32 lanes. Rows are one of 61, so their results are one of 61 (of each expert);
    those against 64 bits, two roundings of bfloat16 (the hidden row's and the result's) and
    sums of 8 terms: 4 u of the terms' size."""
    rows, d, kinds = (1 << 30) + 61 * 500, 8, 61
    gen = torch.Generator().manual_seed(11)
    rn = lambda *s: torch.randn(*s, generator=gen).to(DEV, torch.bfloat16)  # noqa: E731
    small, dsmall = rn(kinds, d), rn(kinds, d)
    chunk = 61 << 16
    of = torch.arange(chunk, device=DEV) % kinds
    x, dy = (torch.empty(rows, d, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    for a in range(0, rows, chunk):
        x[a:a + chunk], dy[a:a + chunk] = small[of[: rows - a]], dsmall[of[: rows - a]]
    n = experts or 1
    ws = [0.4 * rn(n, d, d) for _ in range(3)]
    cuts = [0, 61 * 7_000_000, 61 * 7_000_000, rows] if experts else [0, rows]
    x.requires_grad_(True)
    if experts:
        offsets = torch.tensor(cuts, dtype=torch.int32, device=DEV)
        y = flash_expert_feed_forward(x, offsets, *ws)
    else:
        y = flash_gated_feed_forward(x, *(w[0] for w in ws))
    (dx,) = torch.autograd.grad(y, x, dy)
    for e, (lo, hi) in enumerate(zip(cuts, cuts[1:])):
        if lo == hi:
            continue
        xs, g, u, w = small.double(), ws[0][e].double(), ws[1][e].double(), ws[2][e].double()
        a, b = xs @ g.t(), xs @ u.t()
        s = torch.sigmoid(a)
        h, dh = a * s * b, dsmall.double() @ w
        da, db = dh * b * s * (1 + a * (1 - s)), dh * a * s
        for got, want, size in ((y.detach(), h @ w.t(), h.abs() @ w.abs().t()),
                                (dx, da @ g + db @ u, da.abs() @ g.abs() + db.abs() @ u.abs())):
            assert bool(((got[lo:lo + kinds].double() - want).abs() <= 4 * 2.0 ** -8 * (size + want.abs())).all())
            for at in range(lo, hi, chunk):
                part = got[at:min(at + chunk, hi)]
                assert torch.equal(part, got[lo:lo + kinds][of[: len(part)]])
