"""GPU test of the feed-forward's activations over the whole range of the type."""

import pytest
import torch

from tests._block import TYPES, ffn64, valid_rows

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from flash_spacetime_amd import flash_gated_feed_forward

DEV = "cuda"


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_gates_of_any_size(dtype, act):
    """Projections of up to 1e37 (whose square is infinite) have the activation and the
    derivative of its ends: 0 and 0 below, itself and 1 above. Rows and features are
    one each; single values, rounded a few times: 2^-6 (float32 2^-20)."""
    t, tol = TYPES[dtype], 2.0 ** (-20 if dtype == "f32" else -6)
    gates = [-1e37, -3e30, -1e25, -5e19, -2e19, -1e10, -1e4, 0.0, 1e4, 1e10, 2e19, 5e19, 1e25, 3e30, 1e37]
    for rows in (1, 100, 300):  # the kernel of few rows, and the small tile
        x = torch.zeros(rows, 8, device=DEV, dtype=t)
        x[:, 0] = 1
        for a in gates:
            ws = [torch.zeros(8, 8, device=DEV, dtype=t) for _ in range(3)]
            ws[0][0, 0], ws[1][0, 0], ws[2][0, 0] = a, 0.5, 1
            dy = torch.zeros_like(x)
            dy[-1, 0] = 1
            leaves = [v.detach().requires_grad_(True) for v in (x, *ws)]
            y = flash_gated_feed_forward(*leaves, activation=act)
            got = [y.detach(), *torch.autograd.grad(y, leaves, dy)]
            want = ffn64(x, *ws, None, None, None, act, valid_rows(x.shape, None), dy)
            for g, w in zip(got, want):
                w = w.to(g.device)
                assert bool((g.isfinite() & ((g.double() - w).abs() <= tol * w.abs())).all()), (a, rows)
