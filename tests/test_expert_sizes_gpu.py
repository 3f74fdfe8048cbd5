"""The experts' operators at sizes past those that one launch, or 32 bits, take."""

import pytest
import torch

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from flash_spacetime_amd import flash_expert_route

DEV = "cuda"


@pytest.mark.parametrize("rows,n,k", [((1 << 26) + 777, 129, 1), ((1 << 28) + 4099, 65, 1), ((1 << 29) + 515, 2, 1)])
def test_routes_of_more_rows_than_a_launch_takes(rows, n, k):
    """64, 16 and 8 lanes a row: 2^32 lanes at 2^26, 2^28 and 2^29 rows. Every row holds the
    logits of one of 61, so that what it has to give is the small call's."""
    kinds = torch.randn(61, n, generator=torch.Generator().manual_seed(n)).to(DEV, torch.bfloat16)
    logits = torch.empty(rows, n, device=DEV, dtype=torch.bfloat16)
    chunk = 61 << 20
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
