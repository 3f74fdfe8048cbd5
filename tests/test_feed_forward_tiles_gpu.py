"""GPU parity of the feed-forward's tiles that carry its large calls, against the
definition in 64 bits: contractions of many steps that end inside one, features and
rows that end inside a tile, with and without a list of rows, in every type.

Bounds, in the 2-norm over the exact one's, derived before the first run. u is half a
step of the type. A rounding moves a value by at most u of its power of two, u / sqrt
3 in the root mean square, and over values spread evenly in their logarithm 0.425 u
of the value. In 16-bit types an output takes two of them that count: its own, and
that of the rounded rows it is a sum of (h; da and du), 0.6 u together. 0.66 u is allowed:
a third one (projections kept in 16 bits for the backward) would make 0.74. float32:
sums of up to 2000 products move by sqrt(2000) 2^-24 = 2.7e-6 of their terms' norm at
most, the activation by 1.5e-7; 5e-6 is allowed. Single rows, of few elements, may be
four times as far."""

import ctypes

import pytest
import torch

from tests._block import TYPES, ffn64, valid_rows
from tests._cases import seed_of

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from flash_spacetime_amd import _lib, flash_gated_feed_forward

DEV = "cuda"
NAMES = ("y", "dx", "dw_gate", "dw_up", "dw_down", "db_gate", "db_up", "db_down")
CODES = {"bf16": 0, "f32": 1, "f16": 2}

# rows, D, F; tiles of the gate, output, the projections' gradients, dx and the weights'
# gradients in 16 bits, and in float32
CASES = [
    (16300, 1000, 392, (256, 256, 128, 256, 256), (128,) * 5),
    (16300, 392, 1000, (256, 128, 256, 128, 256), (128,) * 5),
    (12100, 520, 1000, (128, 128, 256, 128, 256), (128,) * 5),
    (2300, 392, 520, (128, 64, 128, 64, 128), (128, 64, 64, 64, 128)),
]


def _tol(dtype):
    return 5e-6 if dtype == torch.float32 else 0.66 * torch.finfo(dtype).eps / 2


def _near(name, got, want, tol):
    got, want = got.detach().double(), want.to(got.device)
    assert got.shape == want.shape, name
    err = float((got - want).norm() / want.norm())
    assert err <= tol, f"{name}: relative error {err:.3e} over {tol:.1e}"
    if got.dim() > 1:
        rows, ref = (got - want).flatten(0, -2).norm(dim=-1), want.flatten(0, -2).norm(dim=-1)
        far = float((rows / (ref + 0.1 * ref.square().mean().sqrt())).max())
        assert far <= 4 * tol, f"{name}: a row's relative error {far:.3e}"


def _make(lead, d, f, dtype, key):
    gen = torch.Generator().manual_seed(seed_of("tiles", key))
    rn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    ws = [(rn(f, d) / d ** 0.5).to(DEV, dtype), (rn(f, d) / d ** 0.5).to(DEV, dtype), (rn(d, f) / f ** 0.5).to(DEV, dtype)]
    bs = [(0.3 * rn(k)).to(DEV, dtype) for k in (f, f, d)]
    return rn(*lead, d).to(DEV, dtype), ws, bs, rn(*lead, d).to(DEV, dtype)


def _tiles(dtype, rows, d, f):
    out = (ctypes.c_int32 * 6)()
    assert _lib.load().fst_ffn_tiles(CODES[dtype], 1, rows, d, f, out) == _lib.FST_OK
    return list(out)


@pytest.mark.parametrize("padded", [False, True], ids=["rows", "padded"])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("case", CASES, ids=lambda c: "x".join(map(str, c[:3])))
def test_tiles_compute(case, dtype, padded):
    rows, d, f, tiles16, tiles32 = case
    assert tuple(_tiles(dtype, rows, d, f)[:5]) == (tiles32 if dtype == "f32" else tiles16)
    t, lead, lens = TYPES[dtype], (rows,), None
    act = ("silu", "gelu", "gelu_tanh")[(d + f + padded) % 3]
    if padded:
        lead = (20, rows // 20)
        lens = torch.randint(0, lead[1] + 1, (20,), generator=torch.Generator().manual_seed(rows))
        lens[3], lens[7], lens[11] = 0, lead[1], 1
    x, ws, bs, dy = _make(lead, d, f, t, (dtype, case[:3], padded))
    valid = valid_rows(x.shape, lens)
    if padded:
        x[~valid.to(DEV)], dy[~valid.to(DEV)] = float("nan"), float("inf")
    leaves = [v.requires_grad_(True) for v in (x, *ws, *bs)]
    y = flash_gated_feed_forward(*leaves, act, seqlens=None if lens is None else lens.to(DEV))
    got = [y, *torch.autograd.grad(y, leaves, dy)]
    if padded:
        assert bool((y[~valid.to(DEV)] == 0).all()) and bool((got[1][~valid.to(DEV)] == 0).all())
    for name, a, b in zip(NAMES, got, ffn64(x, *ws, *bs, act, valid, dy)):
        _near(name, a, b, _tol(t))


@pytest.mark.parametrize("rows,d,f", [(60000, 32, 3848), (60000, 256, 512)])
def test_weight_gradients_of_many_rows_in_float32(rows, d, f):
    """Sums over 60000 rows whose terms have one sign: a run's is one chain, four rows a
    step of the matrix cores; the rounding of the k-th of n additions is at most
    k / n 2^-24 of the whole, over sqrt 3 in the mean square, so a chain's is sqrt(n / 9)
    2^-24, and the runs' own additions and the terms' roundings add 3."""
    t = torch.float32
    x, ws, bs, dy = _make((rows,), d, f, t, ("many", d))
    x, dy = 1 + 0.25 * x, 1 + 0.25 * dy
    leaves = [w.requires_grad_(True) for w in ws]
    got = torch.autograd.grad(flash_gated_feed_forward(x, *leaves, *bs, "silu"), leaves, dy)
    want = ffn64(x, *ws, *bs, "silu", valid_rows(x.shape, None), dy)[2:5]
    steps = rows / _tiles("f32", rows, d, f)[5] / 4
    for name, a, b in zip(NAMES[2:5], got, want):
        err = float((a.double() - b).norm() / b.norm())
        assert err <= ((steps / 9) ** 0.5 + 3) * 2.0 ** -24, (name, err * 2 ** 24)
