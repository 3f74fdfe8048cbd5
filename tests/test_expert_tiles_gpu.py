"""GPU parity of the experts' products in every tile that is compiled for them, against the
definition in 64 bits: contractions of many steps that end inside one, features and runs that
end inside a tile, uneven and empty runs, rows before the first run and behind the last.

Bounds as test_feed_forward_tiles_gpu.py's (the roundings are the same ones): 0.66 u in
the 2-norm in 16-bit types, 5e-6 in float32, single rows four times as far.
"""

import ctypes

import pytest
import torch

from tests._block import TYPES
from tests._cases import seed_of
from tests._experts import expert_ffn64

pytestmark = pytest.mark.gpu

from flash_spacetime_amd import _lib, flash_expert_feed_forward  # noqa: E402

DEV = "cuda"
NAMES = ("y", "dx", "dw_gate", "dw_up", "dw_down")
CODES = {"bf16": 0, "f32": 1, "f16": 2}

# rows, experts, D, F; tiles of the gate, output, the projections' gradients, dx, the weights'
# gradients, and the latter's pieces (1, or more), in 16 bits and in float32
CASES = [
    (50, 1, 136, 1400, (16, 16, 16, 16, 128, 1), (16, 16, 16, 16, 128, 1)),
    (60, 8, 392, 1400, (16, 16, 16, 16, 256, 1), (16, 16, 16, 16, 128, 1)),
    (700, 64, 264, 520, (64, 64, 128, 64, 128, 1), (16, 16, 16, 16, 128, 1)),
    (1500, 3, 136, 1000, (128, 64, 128, 64, 128, 1), (128, 64, 64, 64, 128, 1)),
    (3000, 6, 1000, 520, (128, 128, 128, 128, 128, 1), (128, 128, 64, 128, 128, 1)),
    (3000, 6, 1000, 1000, (128, 128, 128, 128, 256, 1), (64, 128, 128, 128, 128, 1)),
    (9000, 3, 136, 264, (128, 64, 128, 64, 128, 8), (64, 64, 64, 64, 128, 11)),
    (9000, 32, 1032, 392, (128, 256, 256, 256, 256, 1), (64, 64, 64, 64, 128, 1)),
    (16000, 3, 136, 520, (128, 128, 256, 128, 256, 9), (64, 64, 64, 64, 128, 19)),
    (20000, 12, 392, 264, (256, 128, 128, 128, 128, 1), (64, 64, 64, 64, 128, 4)),
    (30000, 16, 392, 392, (256, 256, 256, 256, 256, 1), (64, 64, 64, 64, 128, 3)),
    (30000, 1, 392, 520, (128, 256, 256, 256, 256, 22), (64, 64, 64, 64, 128, 46)),
]


def tiles(dtype, rows, experts, d, f):
    out = (ctypes.c_int32 * 6)()
    assert _lib.load().fst_expert_ffn_tiles(CODES[dtype], rows, experts, d, f, out) == _lib.FST_OK
    return tuple(out)


def _loads(rows, n):
    """Uneven runs, some without rows, one of a single row."""
    share = [0 if i % 5 == 3 else 1 + (i * 7) % 11 for i in range(n)]
    loads = [rows * s // sum(share) for s in share]
    if n > 4:
        loads[1] = 1
    return loads


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c[:4])))
def test_tiles_compute(case, dtype):
    rows, n, d, f, *want_tiles = case
    assert tiles(dtype, rows, n, d, f) == want_tiles[dtype == "f32"]
    t, act = TYPES[dtype], ("silu", "gelu", "gelu_tanh")[(d + f + n) % 3]
    gen = torch.Generator().manual_seed(seed_of("expert tiles", dtype, case[:4]))
    rn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    x, dy = rn(rows, d).to(DEV, t), rn(rows, d).to(DEV, t)
    ws = [(rn(*s) / s[2] ** 0.5).to(DEV, t) for s in ((n, f, d), (n, f, d), (n, d, f))]
    head = rows // 40
    offsets = torch.tensor([head, *_loads(rows - 2 * head, n)]).cumsum(0).int().to(DEV)
    end = int(offsets[-1])
    for v, what in ((x, float("nan")), (dy, float("inf"))):
        v[:head], v[end:] = what, what
    leaves = [v.requires_grad_(True) for v in (x, *ws)]
    y = flash_expert_feed_forward(leaves[0], offsets, *leaves[1:], act)
    got = [y, *torch.autograd.grad(y, leaves, dy)]
    want = expert_ffn64(x, offsets, *ws, act, dy)
    tol = 5e-6 if dtype == "f32" else 0.66 * torch.finfo(t).eps / 2
    for name, a, b in zip(NAMES, got, want):
        a = a.detach().double()
        if name in ("y", "dx"):
            assert bool((a[:head] == 0).all()) and bool((a[end:] == 0).all()), name
        else:
            empty = (offsets[1:] == offsets[:-1]).nonzero()[:, 0]
            assert bool((a[empty] == 0).all()), name
        err = float((a - b).norm() / b.norm())
        assert err <= tol, f"{name}: relative error {err:.3e} over {tol:.1e}"
        far, ref = (a - b).flatten(0, -2).norm(dim=-1), b.flatten(0, -2).norm(dim=-1)
        far = float((far / (ref + 0.1 * ref.square().mean().sqrt())).max())
        assert far <= 4 * tol, f"{name}: a row's relative error {far:.3e}"
