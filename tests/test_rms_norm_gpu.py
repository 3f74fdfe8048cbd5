"""GPU parity of flash_rms_norm and flash_rms_norm_fp8 against their definition in 64 bits.

Bounds, elementwise and derived before the first run. u is half a step of the
output's type, e = 2^-24. rstd: a sum of squares of at most 24 terms a lane and ten
levels of additions, halved by the root, and the root's, the quotient's and the mean's
roundings: at most 32 e. y takes two more products: 64 e of its size cover both.
Each sum of the backward is of the same depth. 8 bits: half a step is 2^-4 of a
normal value, and 2^-10 of the scale below 2^-6 of it.
"""

import pytest
import torch

from tests._block import TYPES, valid_rows
from tests._cases import seed_of
from tests._experts import rms64

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from flash_spacetime_amd import flash_rms_norm, flash_rms_norm_fp8

DEV = "cuda"
E = 2.0 ** -24
EPS = 1e-6


def _u(dtype):
    return torch.finfo(dtype).eps / 2


def _within(name, got, want, bound):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, name
    far = (got - want).abs() - bound
    assert bool((far <= 0).all()), f"{name}: off by {(got - want).abs().max():.3e}, over its bound by {far.max():.3e}"


def _check(x, r, w, seqlens, dy, ds, outs, grads, eps=EPS):
    valid = valid_rows(x.shape, None if seqlens is None else seqlens.cpu())
    y, s, rstd, dx, dw = rms64(x, r, w, eps, valid, dy, ds)
    t, n = x.dtype, x.shape[-1]
    tiny = torch.finfo(t).smallest_normal * torch.finfo(t).eps
    _within("y", outs[0], y, (_u(t) + 64 * E) * y.abs() + tiny)
    if r is not None:
        assert torch.equal(outs[1].detach().double().cpu(), s), "s"
    g = torch.where(valid[..., None], dy.detach().cpu().double(), 0.0).abs()
    wa = torch.ones(n, dtype=torch.float64) if w is None else w.detach().cpu().double().abs()
    xhat, gw = (s * rstd).abs(), g * wa
    bound = _u(t) * dx.abs() + 128 * E * rstd * (gw + xhat * (gw * xhat).mean(-1, keepdim=True)) + 4 * E * dx.abs() + tiny
    if ds is not None:
        bound = bound + 4 * E * torch.where(valid[..., None], ds.detach().cpu().double().abs(), 0.0)
    for name, got in (("dx", grads[0]), ("dresidual", grads[1])):
        if got is not None:
            _within(name, got, dx, bound)
    if grads[2] is not None:
        lead = tuple(range(g.dim() - 1))
        depth = (128 + g[..., 0].numel() / 128) * E  # longest chain of additions, and xhat's own error
        _within("dweight", grads[2], dw, _u(w.dtype) * dw.abs() + depth * (g * xhat).sum(lead) + tiny)


def _run(x, r, w, seqlens, dy, ds, eps=EPS):
    leaves = [t.requires_grad_(True) if t is not None else None for t in (x, r, w)]
    out = flash_rms_norm(leaves[0], leaves[2], eps, residual=leaves[1], seqlens=seqlens)
    outs = out if isinstance(out, tuple) else (out,)
    got = list(torch.autograd.grad(outs, [t for t in leaves if t is not None], (dy, ds) if r is not None else (dy,)))
    return outs, [got.pop(0) if t is not None else None for t in leaves]


def _make(shape, dtype, params, residual, key):
    gen = torch.Generator().manual_seed(seed_of("rms", key))
    rn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    n = shape[-1]
    x = (rn(*shape) * (0.5 + rn(n).abs()) + rn(n)).to(DEV, dtype)
    r = (2 * rn(*shape) + rn(n)).to(DEV, dtype) if residual else None
    w = (1 + 0.3 * rn(n)).to(DEV, params)
    return x, r, w, rn(*shape).to(DEV, dtype), rn(*shape).to(DEV, dtype) if residual else None


WIDTHS = [1, 2, 7, 8, 48, 96, 128, 250, 384, 391, 512, 768, 1000, 1367, 2048, 4096, 6144, 8192, 10007, 16384]


@pytest.mark.parametrize("n", WIDTHS)
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_widths(dtype, n):
    t = TYPES[dtype]
    x, r, w, dy, ds = _make((37, n), t, torch.float32 if n % 2 else t, n % 3 == 0, (dtype, n))
    outs, grads = _run(x, r, w, None, dy, ds)
    _check(x, r, w, None, dy, ds, outs, grads)
    with torch.no_grad():  # the inference call keeps nothing, and gives the same bits
        again = flash_rms_norm(x, w, EPS, residual=r)
        assert torch.equal(again[0] if r is not None else again, outs[0])


@pytest.mark.parametrize("rows", [0, 1, 2, 15, 16, 17, 5000, 40000])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_row_counts(dtype, rows):
    x, r, w, dy, ds = _make((rows, 384), TYPES[dtype], torch.float32, True, (dtype, rows))
    outs, grads = _run(x, r, w, None, dy, ds)
    if rows == 0:
        assert outs[0].shape == outs[1].shape == grads[0].shape == (0, 384)
        assert bool((grads[2] == 0).all())
        return
    _check(x, r, w, None, dy, ds, outs, grads)


@pytest.mark.parametrize("n", [72, 384, 391, 3000])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_padding_is_not_read(dtype, n):
    """Lengths outside 0 .. L are taken within it; what padding holds reaches nothing."""
    t = TYPES[dtype]
    lens = torch.tensor([70, 0, 1, 129, 200, -2, 33])
    x, r, w, dy, ds = _make((7, 129, n), t, torch.float32, True, (dtype, n, "pad"))
    pad = ~valid_rows(x.shape, lens).to(DEV)
    for v, what in ((x, float("nan")), (r, float("inf")), (dy, float("nan")), (ds, -float("inf"))):
        v[pad] = what
    outs, grads = _run(x, r, w, lens.to(DEV), dy, ds)
    assert all(bool((v.detach()[pad] == 0).all()) for v in (*outs, *grads[:2]))
    clean = [torch.where(pad[..., None], 0.0, v.detach()).to(t) for v in (x, r, dy, ds)]
    _check(clean[0], clean[1], w, lens, clean[2], clean[3], outs, grads)
    q, scale, s = flash_rms_norm_fp8(x.detach(), w.detach(), EPS, residual=r.detach(), seqlens=lens.to(DEV))
    assert bool((q.float()[pad] == 0).all()) and bool((scale[pad] == 0).all()) and torch.equal(s, outs[1])


@pytest.mark.parametrize("n", WIDTHS)
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_8_bits(dtype, n):
    t = TYPES[dtype]
    residual = n % 2 == 0
    x, r, w, _, _ = _make((41, n), t, t if n % 3 else torch.float32, residual, (dtype, n, 8))
    x[3] = 0
    if residual:
        r[3] = 0
    out = flash_rms_norm_fp8(x, w, EPS, residual=r)
    y, s, _ = rms64(x, r, w, EPS, valid_rows(x.shape, None))
    q, scale = out[0].double().cpu(), out[1].double().cpu()
    assert out[0].dtype == torch.float8_e4m3fn and out[1].dtype == torch.float32 and out[1].shape == (41,)
    if residual:
        assert torch.equal(out[2].double().cpu(), s)
    want = y.abs().amax(-1) / 448
    live = torch.arange(41) != 3
    assert bool(((scale - want).abs() <= 68 * E * want)[live].all()) and float(scale[3]) == 2.0 ** -126
    assert bool((q.abs().amax(-1) == 448)[live].all()) and bool((q[3] == 0).all())
    _within("q scale", q * scale[:, None], y, (2.0 ** -4 + 2.0 ** -12) * y.abs() + 1.01 * 2.0 ** -10 * scale[:, None])


def test_rows_that_are_not_finite():
    """NaN and infinities stay in their rows; small and large rows keep their digits."""
    x, _, w, _, _ = _make((6, 384), torch.float32, torch.float32, False, "odd rows")
    x[0, 5], x[1, 7] = float("nan"), float("inf")
    x[2] *= 1e-30
    x[3] *= 1e15
    for got in (flash_rms_norm(x, w), flash_rms_norm_fp8(x, w)[0].float()):
        assert bool(got[0].isnan().all()) and bool(got[1, 7].isnan()) and bool((got[1].nan_to_num() == 0).all())
        assert bool(got[2:].isfinite().all())
    y, _, _ = rms64(x[2:], None, w, 1e-6, valid_rows((4, 384), None))
    _within("y", flash_rms_norm(x, w)[2:], y, 65 * E * y.abs() + 2.0 ** -149)
    q, scale = flash_rms_norm_fp8(x[2:], w)
    _within("q", q.double() * scale.double()[:, None], y, 0.0626 * y.abs() + 1.01 * 2.0 ** -10 * scale.double().cpu()[:, None])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_strides(dtype):
    """Slices, transposed and expanded rows give the dense call's bits."""
    t = TYPES[dtype]
    x, r, w, dy, ds = _make((6, 50, 384), t, torch.float32, True, (dtype, "strides"))
    want = _run(x.clone(), r.clone(), w.clone(), None, dy, ds)
    wide = torch.zeros(6, 50, 400, device=DEV, dtype=t)
    wide[..., 9:393] = x.detach()
    turned = r.detach().permute(1, 0, 2).contiguous().permute(1, 0, 2)
    got = _run(wide[..., 9:393].detach(), turned.detach(), w.clone(), None, dy.permute(1, 0, 2).contiguous().permute(1, 0, 2), ds)
    for a, b in zip((*want[0], *want[1]), (*got[0], *got[1])):
        assert torch.equal(a, b)
    q = flash_rms_norm_fp8(x.detach(), w.detach(), residual=r.detach())
    p = flash_rms_norm_fp8(wide[..., 9:393], w.detach(), residual=turned)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(q, p))
    one = dy[:1, :1].expand(6, 50, 384)  # a broadcast gradient
    a = _run(x.detach(), r.detach(), w.detach(), None, one, ds)
    b = _run(x.detach(), r.detach(), w.detach(), None, one.contiguous(), ds)
    assert all(torch.equal(i, j) for i, j in zip(a[1], b[1]))


def test_single_gradients_and_unused_outputs():
    x, r, w, dy, ds = _make((40, 256), torch.bfloat16, torch.float32, True, "single")
    full = _run(x, r, w, None, dy, ds)[1]
    for i in range(3):
        leaves = [t.detach().requires_grad_(i == j) for j, t in enumerate((x, r, w))]
        out = flash_rms_norm(leaves[0], leaves[2], EPS, residual=leaves[1])
        assert torch.equal(torch.autograd.grad(out, leaves[i], (dy, ds))[0], full[i])
    xs = x.detach().requires_grad_(True)
    y, s = flash_rms_norm(xs, w.detach(), EPS, residual=r.detach())
    assert torch.equal(torch.autograd.grad(s, xs, ds)[0], ds)


def test_gradient_against_differences():
    x, r, w, dy, _ = _make((3, 40), torch.float32, torch.float32, False, "diff")
    dy = dy.double().cpu()
    (_, grads), h = _run(x, None, w, None, dy.float().to(DEV), None), 1e-5
    f = lambda a, b: float((rms64(a, None, b, EPS, valid_rows(a.shape, None))[0] * dy).sum())  # noqa: E731
    x64, w64 = x.detach().double().cpu(), w.detach().double().cpu()
    for at in ((0, 0), (1, 17), (2, 39)):
        d = torch.zeros_like(x64)
        d[at] = h
        slope = (f(x64 + d, w64) - f(x64 - d, w64)) / (2 * h)
        assert abs(slope - float(grads[0][at])) <= 1e-5 * max(1.0, abs(slope))
    d = torch.zeros_like(w64)
    d[11] = h
    assert abs((f(x64, w64 + d) - f(x64, w64 - d)) / (2 * h) - float(grads[2][11])) <= 1e-5 * 20


def test_replays_in_a_graph():
    """Captured calls, forward, backward and 8 bits, follow their inputs at every replay."""
    x, r, w, dy, ds = _make((8, 40, 384), torch.bfloat16, torch.float32, True, "graph")
    lens = torch.tensor([40, 3, 0, 17, 22, 40, 1, 9], device=DEV, dtype=torch.int32)

    def step():
        outs, grads = _run(x.detach(), r.detach(), w.detach(), lens, dy, ds)
        q, scale, _ = flash_rms_norm_fp8(x.detach(), w.detach(), residual=r.detach(), seqlens=lens)
        return [*(o.detach() for o in outs), *grads, scale, q.view(torch.uint8)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
    for i in range(3):
        x.data.mul_(-1.25)
        lens.copy_(torch.roll(lens, 1))
        for t in static:
            t.fill_(3)
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(static, want):
            assert torch.equal(a, c), f"replay {i}"


def test_autocast():
    x, r, w, _, _ = _make((20, 256), torch.float32, torch.float32, True, "autocast")
    with torch.autocast("cuda", torch.bfloat16):
        y, s = flash_rms_norm(x.bfloat16(), w, residual=r)
        assert y.dtype == s.dtype == torch.float32
        assert flash_rms_norm(x.bfloat16(), w.half()).dtype == torch.bfloat16
        assert flash_rms_norm_fp8(x.bfloat16(), w, residual=r)[2].dtype == torch.float32


def test_refusals():
    x, w = torch.randn(4, 16, device=DEV), torch.ones(16, device=DEV)
    for f in (flash_rms_norm, flash_rms_norm_fp8):
        with pytest.raises(ValueError, match="bfloat16"):
            f(x.double())
        with pytest.raises(ValueError, match="weight must be"):
            f(x, w[:8])
        with pytest.raises(ValueError, match="weight must be"):
            f(x, w.half())
        with pytest.raises(ValueError, match="residual"):
            f(x, w, residual=x[:2])
        with pytest.raises(ValueError, match="eps"):
            f(x, w, -1.0)
        with pytest.raises(ValueError, match="seqlens"):
            f(x, w, seqlens=torch.tensor([1, 2], device=DEV))
        with pytest.raises(ValueError, match="16384"):
            f(torch.zeros(1, 16385, device=DEV))
        with pytest.raises(RuntimeError, match="GPU"):
            f(x, w.cpu())
    with pytest.raises(ValueError, match="no derivative"):
        flash_rms_norm_fp8(x, w.requires_grad_(True))
    with torch.no_grad():
        flash_rms_norm_fp8(x, w)


def test_rows_past_32_bits():
    """280000 rows of 8192: element offsets of the last rows pass 2^31."""
    rows, n = 280_000, 8192
    x = torch.empty(rows, n, device=DEV, dtype=torch.bfloat16)
    x.copy_((1 + torch.arange(rows, device=DEV) % 63)[:, None] * (1 + torch.arange(n, device=DEV) % 3)[None, :])
    x.requires_grad_(True)
    y = flash_rms_norm(x)
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    q, scale = flash_rms_norm_fp8(x.detach())
    for at in (0, 131_071, 262_143, 262_145, rows - 1):
        row = x.detach()[at:at + 1].clone()
        want = _run(row, None, None, None, torch.ones_like(row), None)
        assert torch.equal(y.detach()[at:at + 1], want[0][0].detach()) and torch.equal(dx[at:at + 1], want[1][0])
        one = flash_rms_norm_fp8(row.detach())
        assert torch.equal(q[at:at + 1].float(), one[0].float()) and torch.equal(scale[at:at + 1], one[1])
