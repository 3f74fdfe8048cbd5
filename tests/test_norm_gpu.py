"""GPU parity of flash_layer_norm against its definition in 64 bits.

Bounds, elementwise and derived before the first run. u is half a step of the
output's type, e = 2^-24. The kernel's float32 arithmetic moves a normalised
value by a few e times the magnitudes it is formed from: the mean and variance
of a row are sums of at most 16 terms a lane, a few lanes' tree and one
correction, each bounded by 64 e of the sum of the terms' magnitudes.
"""

import pytest
import torch

from tests._block import TYPES, norm64, valid_rows
from tests._cases import seed_of

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from flash_spacetime_amd import flash_layer_norm

DEV = "cuda"
E = 2.0 ** -24
EPS = 1e-5


def _u(dtype):
    return torch.finfo(dtype).eps / 2


def _within(name, got, want, bound):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, name
    far = (got - want).abs() - bound
    assert bool((far <= 0).all()), f"{name}: off by {(got - want).abs().max():.3e}, over its bound by {far.max():.3e}"


def _check(x, r, w, b, seqlens, dy, ds, outs, grads, eps=EPS):
    """outs: y (and s); grads of x, r, w, b (None where absent)."""
    valid = valid_rows(x.shape, None if seqlens is None else seqlens.cpu())
    y, s, dx, dw, db = norm64(x.detach(), None if r is None else r.detach(), w, b, eps, valid, dy, ds)
    t, n = x.dtype, x.shape[-1]
    tiny = torch.finfo(t).smallest_normal * torch.finfo(t).eps  # a denormal step
    wa = torch.ones(n, dtype=torch.float64) if w is None else w.detach().cpu().double().abs()
    ba = torch.zeros(n, dtype=torch.float64) if b is None else b.detach().cpu().double().abs()
    m = s.mean(-1, keepdim=True)
    rstd = ((s - m).square().mean(-1, keepdim=True) + eps).rsqrt()
    xhat = ((s - m) * rstd).abs()
    # xhat: its own rounding and the mean's, which the kernel corrects to e of the row's magnitude
    ex = 64 * E * (xhat + 1) + 4 * E * s.abs().mean(-1, keepdim=True) * rstd
    _within("y", outs[0], y, _u(t) * y.abs() + (1 + _u(t)) * (ex * wa + 4 * E * ba) + tiny)
    if r is not None:
        assert torch.equal(outs[1].detach().double().cpu(), s), "s"
    g = torch.where(valid[..., None], dy.detach().cpu().double(), 0.0)
    gw = g.abs() * wa
    mean = lambda v: v.mean(-1, keepdim=True)  # noqa: E731
    # dx: each term's relative error, and xhat's error in the two places it stands
    stat = 2 * E * m.abs() * rstd  # the saved mean is rounded once
    eg = 64 * E * (gw + mean(gw) + xhat * mean(gw * xhat)) + (ex + stat) * mean(gw * xhat) + xhat * mean(gw * (ex + stat))
    bound = _u(t) * dx.abs() + 2 * rstd * eg + 4 * E * dx.abs() + tiny
    if ds is not None:
        bound = bound + 4 * E * ds.detach().cpu().double().abs()
    for name, got in (("dx", grads[0]), ("dresidual", grads[1])):
        if got is not None:
            _within(name, got, dx, bound)
    lead = tuple(range(g.dim() - 1))
    rows = g[..., 0].numel()
    depth = (64 + rows / 128) * E  # longest chain of additions
    if grads[2] is not None:
        terms = (g.abs() * xhat).sum(lead)
        _within("dweight", grads[2], dw, _u(w.dtype) * dw.abs() + depth * terms + (g.abs() * (ex + stat)).sum(lead) + tiny)
    if grads[3] is not None:
        _within("dbias", grads[3], db, _u(b.dtype) * db.abs() + depth * g.abs().sum(lead) + tiny)


def _run(x, r, w, b, seqlens, dy, ds, eps=EPS):
    leaves = [t.requires_grad_(True) if t is not None else None for t in (x, r, w, b)]
    out = flash_layer_norm(*(leaves[0], leaves[2], leaves[3]), eps, residual=leaves[1], seqlens=seqlens)
    outs = out if isinstance(out, tuple) else (out,)
    used = [t for t in leaves if t is not None]
    got = list(torch.autograd.grad(outs, used, (dy, ds) if r is not None else (dy,)))
    return outs, [got.pop(0) if t is not None else None for t in leaves]


def _make(shape, dtype, params, residual, key):
    gen = torch.Generator().manual_seed(seed_of("norm", key))
    rn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    n = shape[-1]
    x = (rn(*shape) * (0.5 + rn(n).abs()) + rn(n)).to(DEV, dtype)
    r = (2 * rn(*shape) + rn(n)).to(DEV, dtype) if residual else None
    w, b = ((1 + 0.3 * rn(n)).to(DEV, params), (0.2 * rn(n)).to(DEV, params))
    dy = rn(*shape).to(DEV, dtype)
    ds = rn(*shape).to(DEV, dtype) if residual else None
    return x, r, w, b, dy, ds


@pytest.mark.parametrize("n", [1, 2, 7, 8, 48, 96, 128, 250, 384, 391, 512, 768, 1000, 1367, 2048, 4096, 6144, 8192, 10007,
                               16384])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_widths(dtype, n):
    t = TYPES[dtype]
    params = torch.float32 if n % 2 else t
    residual = n % 3 == 0
    case = _make((37, n), t, params, residual, (dtype, n))
    x, r, w, b, dy, ds = case
    outs, grads = _run(x, r, w, b, None, dy, ds)
    _check(x, r, w, b, None, dy, ds, outs, grads)


@pytest.mark.parametrize("rows", [0, 1, 2, 15, 16, 17, 5000, 40000])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_row_counts(dtype, rows):
    t = TYPES[dtype]
    x, r, w, b, dy, ds = _make((rows, 384), t, torch.float32, True, (dtype, rows))
    outs, grads = _run(x, r, w, b, None, dy, ds)
    if rows == 0:
        assert outs[0].shape == outs[1].shape == grads[0].shape == (0, 384)
        assert bool((grads[2] == 0).all()) and bool((grads[3] == 0).all())
        return
    _check(x, r, w, b, None, dy, ds, outs, grads)


@pytest.mark.parametrize("n", [40, 384, 391, 3000])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_padded_batches_ignore_what_padding_holds(dtype, residual, n):
    """Padding rows of every input hold NaN and infinities; an event of no
    tokens, one past the padded length (taken as that) and a negative length."""
    t = TYPES[dtype]
    lens = torch.tensor([9, 0, 33, 1, 40, -3], dtype=torch.int64)
    x, r, w, b, dy, ds = _make((6, 33, n), t, torch.float32, residual, (dtype, n, "pad"))
    valid = valid_rows(x.shape, lens)
    junk = torch.tensor([float("nan"), float("inf"), -float("inf")], device=DEV)
    fill = junk[torch.arange(n, device=DEV) % 3].to(t)
    for m in (x, r, dy, ds):
        if m is not None:
            m[~valid.to(DEV)] = fill
    outs, grads = _run(x, r, w, b, lens.to(DEV), dy, ds)
    for o in (*outs, *(g for g in grads[:2] if g is not None)):
        assert bool((o.detach()[~valid.to(DEV)] == 0).all())
    z = lambda m: None if m is None else torch.where(valid[..., None].to(DEV), m.detach(), torch.zeros_like(m))  # noqa: E731
    _check(z(x), z(r), w, b, lens, z(dy), z(ds), outs, grads)


def test_all_events_empty():
    x, r, w, b, dy, ds = _make((4, 5, 64), torch.bfloat16, torch.float32, True, "empty")
    outs, grads = _run(x, r, w, b, torch.zeros(4, dtype=torch.int32, device=DEV), dy, ds)
    for t in (*outs, *grads):
        assert bool((t == 0).all())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("view", ["row_stride", "columns", "transposed", "offset", "expanded", "heads"])
def test_strides_and_alignments(dtype, view):
    t = TYPES[dtype]
    n, rows = 200, 24
    gen = torch.Generator().manual_seed(seed_of("strides", dtype, view))
    rn = lambda *s: torch.randn(*s, generator=gen).to(DEV, t)  # noqa: E731

    def make():
        if view == "row_stride":
            return rn(rows, 3 * n)[:, n:2 * n]
        if view == "columns":
            return rn(rows, n, 2)[..., 1]
        if view == "transposed":
            return rn(n, rows).t()
        if view == "offset":
            return rn(rows * n + 1)[1:].view(rows, n)
        if view == "expanded":
            return rn(1, n).expand(rows, n)
        return rn(2, 12, 3, n)[:, :, 1]  # heads of a packed projection: [2, 12, n]

    x, r, dy, ds = make(), make(), make(), make()
    w, b = rn(n).float(), rn(n + 1).float()[1:]
    leaf = x.detach().requires_grad_(True)
    rleaf = r.detach().requires_grad_(True)
    wl, bl = w.clone().requires_grad_(True), b.detach().requires_grad_(True)
    y, s = flash_layer_norm(leaf, wl, bl, EPS, residual=rleaf)
    grads = torch.autograd.grad((y, s), (leaf, rleaf, wl, bl), (dy, ds))
    _check(x, r, w, b, None, dy, ds, (y, s), grads)


def test_optional_parameters_and_gradients():
    """No weight, no bias, either alone; frozen leaves; an unused output."""
    x, r, w, b, dy, ds = _make((50, 96), torch.float32, torch.float32, True, "optional")
    for ww, bb in ((None, None), (w, None), (None, b)):
        outs, grads = _run(x.detach(), None, None if ww is None else ww.detach(), None if bb is None else bb.detach(),
                           None, dy, None)
        _check(x, None, ww, bb, None, dy, None, outs, grads)
    x, w, b = x.detach(), w.detach(), b.detach()
    y = flash_layer_norm(x.requires_grad_(True), w, b)
    assert torch.autograd.grad(y, x, dy)[0].shape == x.shape
    x = x.detach()
    y = flash_layer_norm(x, w.requires_grad_(True), b)
    (dw,) = torch.autograd.grad(y, w, dy)
    valid = valid_rows(x.shape, None)
    want = norm64(x, None, w, b, EPS, valid, dy)[3]
    assert float((dw.double().cpu() - want).abs().max()) <= 1e-4
    # only the sum's gradient: it passes through unchanged
    xl = x.clone().requires_grad_(True)
    _, s = flash_layer_norm(xl, w.detach(), b, residual=r)
    assert torch.equal(torch.autograd.grad(s, xl, ds)[0], ds)
    # only y's
    rl = r.clone().requires_grad_(True)
    y, _ = flash_layer_norm(x, w.detach(), b, residual=rl)
    want = norm64(x, r, w, b, EPS, valid, dy)[2]
    assert float((torch.autograd.grad(y, rl, dy)[0].double().cpu() - want).abs().max()) <= 1e-4


def test_one_tensor_in_two_places_and_a_graph_run_twice():
    """The residual is x itself, weight and bias are one; the graph is kept."""
    x, _, w, _, dy, ds = _make((37, 391), torch.bfloat16, torch.float32, True, "shared")
    outs, (dx, dr, dw, db) = _run(x, x.clone(), w, w.clone(), None, dy, ds)
    a, p = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    y, s = flash_layer_norm(a, p, p, residual=a)
    assert torch.equal(y, outs[0]) and torch.equal(s, outs[1])
    for keep in (True, False):
        ga, gp = torch.autograd.grad((y, s), (a, p), (dy, ds), retain_graph=keep)
        assert torch.equal(ga, dx + dr) and torch.equal(gp, dw + db)


def test_rows_do_not_touch_each_other():
    """A row of NaN, one of infinities and one of the type's lowest value leave
    the others' bits alone; a constant row comes back as the bias."""
    gen = torch.Generator().manual_seed(5)
    x = torch.randn(20, 384, generator=gen).to(DEV, torch.bfloat16)
    b = torch.randn(384, generator=gen).to(DEV)
    clean = flash_layer_norm(x, None, b)
    y = x.clone()
    y[3], y[7], y[11], y[15] = float("nan"), float("inf"), torch.finfo(torch.bfloat16).min, 2.5
    got = flash_layer_norm(y, None, b)
    keep = [i for i in range(20) if i not in (3, 7, 11, 15)]
    assert torch.equal(got[keep], clean[keep])
    assert bool(got[3].isnan().all()) and bool(got[7].isnan().all())
    assert torch.equal(got[15], b.to(torch.bfloat16))


@pytest.mark.parametrize("mean", [0.0, 1e3, 1e5])
def test_mean_far_from_zero(mean):
    """float32 rows whose mean is large beside their spread: the deviations are
    exact differences, so what is left is one part in 2^24 of them."""
    gen = torch.Generator().manual_seed(11)
    x = (torch.randn(64, 1000, generator=gen) + mean).to(DEV)
    y = flash_layer_norm(x)
    want, _ = norm64(x, None, None, None, EPS, valid_rows(x.shape, None))
    # the first mean is rounded to e mean; its square is all that is lost of the variance
    tol = 64 * E * 8 + (mean * E) ** 2
    assert float((y.double().cpu() - want).abs().max()) <= tol


def test_gradient_against_differences():
    gen = torch.Generator().manual_seed(21)
    rn = lambda *s: torch.randn(*s, generator=gen).to(DEV)  # noqa: E731
    x, w, b, c = rn(6, 70), rn(70), rn(70), rn(6, 70)
    loss = lambda *a: float((flash_layer_norm(*a, 1e-5).double() * c.double()).sum())  # noqa: E731
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(flash_layer_norm(*leaves, 1e-5), leaves, c)
    h = 2.0 ** -7
    for i, g in enumerate(grads):
        v = rn(*g.shape)
        at = lambda k: loss(*(t + k * h * v if j == i else t for j, t in enumerate((x, w, b))))  # noqa: E731
        # fourth-order difference: 420 outputs of order 1 to 3, each off by about 1e-6, over 12 h, and h^4 terms
        got = (8 * (at(1) - at(-1)) - (at(2) - at(-2))) / (12 * h)
        want = float((g.double() * v.double()).sum())
        scale = float(g.double().norm() * v.double().norm())
        assert abs(got - want) <= 2e-3 * scale, (i, got, want)


def test_bitwise_repeatable_and_on_another_stream():
    x, r, w, b, dy, ds = _make((3000, 384), torch.bfloat16, torch.float32, True, "repeat")
    outs, grads = _run(x, r, w, b, None, dy, ds)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs2, grads2 = _run(x.detach(), r.detach(), w.detach(), b.detach(), None, dy, ds)
    side.synchronize()
    for a, c in zip((*outs, *grads), (*outs2, *grads2)):
        assert torch.equal(a, c)


def test_replays_in_a_graph():
    x, r, w, b, dy, ds = _make((8, 40, 384), torch.bfloat16, torch.float32, True, "graph")
    lens = torch.tensor([40, 3, 0, 17, 22, 40, 1, 9], device=DEV, dtype=torch.int32)

    def step():
        outs, grads = _run(x.detach(), r.detach(), w.detach(), b.detach(), lens, dy, ds)
        return [*(o.detach() for o in outs), *grads]

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
            t.fill_(float("nan"))
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for a, c in zip(static, want):
            assert torch.equal(a, c), f"replay {i}"


def test_double_backward_and_stale_inputs_are_refused():
    """Only first derivatives are offered, and an input modified in place after
    the forward is noticed, through the host extension and without it."""
    x = torch.randn(4, 32, device=DEV, requires_grad=True)
    g = torch.autograd.grad(flash_layer_norm(x).square().sum(), x, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="twice"):
        g.sum().backward()
    z = x.detach().clone().requires_grad_(True) * 1.0
    y = flash_layer_norm(z)
    z.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_host_extension_and_python_path_agree_bitwise(monkeypatch, dtype, residual):
    from flash_spacetime_amd import _lib

    assert _lib.host() is not None
    lens = torch.tensor([5, 0, 12], device=DEV)
    for key, shape, sl in (("rows", (33, 72), None), ("pad", (3, 12, 391), lens), ("one", (384,), None)):
        x, r, w, b, dy, ds = _make(shape, TYPES[dtype], torch.float32, residual, (dtype, key))
        a = _run(x, r, w, b, sl, dy, ds)
        with monkeypatch.context() as m:
            m.setattr(_lib, "host", lambda: None)
            c = _run(x.detach(), None if r is None else r.detach(), w.detach(), b.detach(), sl, dy, ds)
        for p, q in zip((*a[0], *a[1]), (*c[0], *c[1])):
            assert (p is None) == (q is None) and (p is None or torch.equal(p, q))


def test_saved_tensor_hooks_see_what_the_backward_keeps():
    x = torch.randn(6, 64, device=DEV, requires_grad=True)
    seen = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: seen.append(tuple(t.shape)) or t.cpu(), lambda t: t.to(DEV)):
        y = flash_layer_norm(x)
    assert (6, 64) in seen and (6, 2) in seen
    dy = torch.randn_like(y)
    want = torch.autograd.grad(flash_layer_norm(x), x, dy)[0]
    assert torch.equal(torch.autograd.grad(y, x, dy)[0], want)


def test_refusals():
    x = torch.randn(2, 3, 16, device=DEV)
    w = torch.randn(16, device=DEV)
    bad = [
        (dict(x=x.double()), "bfloat16"), (dict(weight=w[:8]), "weight"), (dict(weight=w.double()), "float32"),
        (dict(weight=w, bias=w.half()), "bias"), (dict(x=x.half(), weight=w, bias=w.half()), "share"),
        (dict(residual=x[:1]), "residual"), (dict(residual=x.half()), "residual"), (dict(eps=-1.0), "eps"),
        (dict(seqlens=torch.tensor([1, 2, 3], device=DEV)), "seqlens"), (dict(seqlens=torch.tensor([1.0, 2.0], device=DEV)), "integer"),
        (dict(x=x[0], seqlens=torch.tensor([1, 2], device=DEV)), "padded"), (dict(x=torch.zeros(2, 0, device=DEV)), "features"),
        (dict(x=torch.zeros(1, 16385, device=DEV)), "16384"),
    ]
    for kwargs, what in bad:
        call = {"x": x, **kwargs}
        with pytest.raises(ValueError, match=what):
            flash_layer_norm(**call)
    with pytest.raises(RuntimeError, match="GPU"):
        flash_layer_norm(x, w.cpu())
    # lengths on the host are moved; the defaults are those of the docstring
    y = flash_layer_norm(x, seqlens=torch.tensor([1, 2]))
    assert bool((y[0, 1:] == 0).all()) and bool((y[1, :2] != 0).any())
