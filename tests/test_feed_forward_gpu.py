"""GPU parity of flash_gated_feed_forward against its definition in 64 bits.

Bounds, in the 2-norm of an output over the exact one's, derived before the
first run. 16-bit types (u half a step): an output takes its own rounding, the
rounding of the hidden rows or of the gradients of both projections, and in the
backward the roundings of the saved projections; independent relative errors
of at most u, and for the gate's derivative a factor of at most about one: five
of them at u / sqrt 3 rms each are 1.3 u, and 2 u = eps is allowed. float32: sums
of up to 1500 products take about sqrt(1500) 2^-24 = 2.3e-6 of the terms' norm,
and the activation 1.5e-7; 5e-6 is allowed. Single rows, of few elements, may be
four times as far.
"""

import pytest
import torch

from tests._block import TYPES, ffn64, valid_rows
from tests._cases import seed_of

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from flash_spacetime_amd import flash_gated_feed_forward

DEV = "cuda"
NAMES = ("y", "dx", "dw_gate", "dw_up", "dw_down", "db_gate", "db_up", "db_down")


def _tol(dtype):
    return 5e-6 if dtype == torch.float32 else torch.finfo(dtype).eps


def _near(name, got, want, tol):
    got, want = got.detach().double(), want.to(got.device)
    assert got.shape == want.shape, name
    err = float((got - want).norm() / want.norm().clamp_min(1e-30))
    assert err <= tol, f"{name}: relative error {err:.3e} over {tol:.1e}"
    if got.dim() > 1:
        rows, ref = (got - want).flatten(0, -2).norm(dim=-1), want.flatten(0, -2).norm(dim=-1)
        typical = ref.square().mean().sqrt()
        far = float((rows / (ref + 0.1 * typical).clamp_min(1e-30)).max())
        assert far <= 4 * tol, f"{name}: a row's relative error {far:.3e}"


def _make(lead, d, f, dtype, biases, key):
    gen = torch.Generator().manual_seed(seed_of("ffn", key))
    rn = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    x = rn(*lead, d).to(DEV, dtype)
    ws = [(rn(f, d) / d ** 0.5).to(DEV, dtype), (rn(f, d) / d ** 0.5).to(DEV, dtype), (rn(d, f) / f ** 0.5).to(DEV, dtype)]
    bs = [(0.3 * rn(k)).to(DEV, dtype) if biases else None for k in (f, f, d)]
    return x, ws, bs, rn(*lead, d).to(DEV, dtype)


def _run(x, ws, bs, act, seqlens, dy):
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (x, *ws, *bs)]
    y = flash_gated_feed_forward(*leaves, act, seqlens=seqlens)
    got = list(torch.autograd.grad(y, [t for t in leaves if t is not None], dy))
    return [y, *(got.pop(0) if t is not None else None for t in leaves)]


def _compare(got, want, dtype):
    for name, a, b in zip(NAMES, got, want):
        if a is not None:
            _near(name, a, b, _tol(dtype))


SIZES = [(1, 8, 8), (3, 16, 24), (17, 32, 64), (64, 64, 128), (65, 40, 72), (127, 72, 136), (129, 200, 264), (187, 384, 1024),
         (300, 136, 520), (513, 96, 1000), (1000, 384, 256), (2050, 768, 320)]


@pytest.mark.parametrize("rows,d,f", SIZES)
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_sizes(dtype, rows, d, f):
    act = ("silu", "gelu", "gelu_tanh")[(rows + d) % 3]
    t = TYPES[dtype]
    x, ws, bs, dy = _make((rows,), d, f, t, f % 16 == 8 or rows == 187, (dtype, rows, d, f))
    got = _run(x, ws, bs, act, None, dy)
    _compare(got, ffn64(x, *ws, *bs, act, valid_rows(x.shape, None), dy), t)
    with torch.no_grad():  # the inference call keeps nothing, and gives the same bits
        assert torch.equal(flash_gated_feed_forward(x, *ws, *bs, act), got[0])


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_padded_batches_ignore_what_padding_holds(dtype, act):
    t = TYPES[dtype]
    lens = torch.tensor([70, 0, 1, 129, 200, -2, 33], dtype=torch.int64)
    x, ws, bs, dy = _make((7, 129), 72, 136, t, True, (dtype, act, "pad"))
    valid = valid_rows(x.shape, lens)
    pad = ~valid.to(DEV)
    x[pad], dy[pad] = float("nan"), float("inf")
    got = _run(x, ws, bs, act, lens.to(DEV), dy)
    assert bool((got[0].detach()[pad] == 0).all()) and bool((got[1][pad] == 0).all())
    _compare(got, ffn64(x, *ws, *bs, act, valid, dy), t)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_padded_equals_packed_bitwise(dtype):
    """The valid rows of a padded call are those of the packed call."""
    t = TYPES[dtype]
    lens = torch.tensor([5, 64, 0, 17, 90])
    x, ws, bs, dy = _make((5, 90), 384, 512, t, True, (dtype, "packed"))
    valid = valid_rows(x.shape, lens).to(DEV)
    a = _run(x, ws, bs, "silu", lens.to(DEV), dy)
    b = _run(x[valid], ws, bs, "silu", None, dy[valid])
    assert torch.equal(a[0][valid], b[0]) and torch.equal(a[1][valid], b[1])


def test_all_events_empty_and_no_rows():
    x, ws, bs, dy = _make((3, 7), 64, 128, torch.bfloat16, True, "empty")
    got = _run(x, ws, bs, "silu", torch.zeros(3, dtype=torch.int32, device=DEV), dy)
    assert all(bool((t == 0).all()) for t in got)
    got = _run(x[:0], ws, bs, "silu", None, dy[:0])
    assert got[0].shape == got[1].shape == (0, 7, 64)
    assert all(bool((t == 0).all()) for t in got[2:])


def test_more_events_than_a_grid_has_workgroups():
    """2^24 events of one row: their padding is zeroed by fewer workgroups."""
    b, t = (1 << 24) + 3, torch.float16
    x, ws, bs, _ = _make((64,), 8, 8, t, True, "events")
    x = x.repeat(b // 64 + 1, 1)[:b].contiguous()
    lens = (torch.arange(b, device=DEV) % 3 != 1).int()
    valid = lens.bool()
    a = _run(x[:, None], ws, bs, "silu", lens, x[:, None])
    p = _run(x[valid], ws, bs, "silu", None, x[valid])
    for got, want in zip(a[:2], p[:2]):
        assert torch.equal(got[:, 0][valid], want) and bool((got[:, 0][~valid] == 0).all())


@pytest.mark.parametrize("lead", [(0, 7), (3, 0)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_padded_batch_without_rows(dtype, lead):
    """No event, or none of any length: the gradients of the weights are zeros,
    whatever the memory that would have held the list of rows holds."""
    x, ws, bs, dy = _make(lead, 64, 128, TYPES[dtype], True, "rowless")
    lens = torch.full((lead[0],), 5, dtype=torch.int32, device=DEV)
    got = _run(x, ws, bs, "silu", lens, dy)
    assert got[0].shape == got[1].shape == (*lead, 64)
    assert all(bool((t == 0).all()) for t in got[2:])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("view", ["row_stride", "odd_stride", "transposed", "offset", "expanded", "batch_first"])
def test_strides_and_alignments(dtype, view):
    t = TYPES[dtype]
    d, f, rows = 72, 136, 40
    x, ws, bs, dy = _make((rows,), d, f, t, True, (dtype, view))

    def see(v):
        if view == "row_stride":
            return torch.cat([v, v, v], 1)[:, d:2 * d]
        if view == "odd_stride":
            return torch.cat([v, v[:, :3]], 1)[:, :d]
        if view == "transposed":
            return v.t().contiguous().t()
        if view == "offset":
            return torch.cat([v.flatten()[:1], v.flatten()])[1:].view(rows, d)
        if view == "expanded":
            return v[:1].expand(rows, d)
        return v.view(4, 10, d).transpose(0, 1)

    x, dy = see(x), see(dy)
    ws = [w.t().contiguous().t() for w in ws]
    bs = [torch.cat([b[:1], b])[1:] for b in bs]
    got = _run(x, ws, bs, "gelu", None, dy)
    _compare(got, ffn64(x, *ws, *bs, "gelu", valid_rows(x.shape, None), dy), t)


def test_subsets_of_gradients():
    x, ws, bs, dy = _make((150,), 64, 96, torch.float32, True, "subset")
    full = _run(x, ws, bs, "silu", None, dy)
    tensors = [x, *ws, *bs]
    for need in ([0], [1], [2], [3], [4], [5], [6], [0, 3], [1, 2, 6]):
        leaves = [t.detach().requires_grad_(i in need) for i, t in enumerate(tensors)]
        y = flash_gated_feed_forward(*leaves)
        for i, g in zip(need, torch.autograd.grad(y, [leaves[i] for i in need], dy)):
            assert torch.equal(g, full[1 + i]), NAMES[1 + i]


def test_bias_gradients_of_many_rows_in_float32():
    """60000 rows beside weights of many tiles, whose runs of rows are long. A column
    goes through chains of 64 additions (256 rows, four at a time), at most 235 (the
    sums of 256 rows of all runs together) and one; the rounding of the k-th of n is
    at most k / n 2^-24 of the whole, over sqrt 3 in the mean square, so a chain's is
    sqrt(n / 9) 2^-24 and all of them sqrt(300 / 9) = 5.8. (One chain over each run
    gave 6.5.)"""
    x, ws, bs, dy = _make((60000,), 32, 3848, torch.float32, True, "many")
    b = bs[2].detach().requires_grad_(True)
    dy = 1 + 0.25 * dy
    got, = torch.autograd.grad(flash_gated_feed_forward(x, *ws, *bs[:2], b, "silu"), b, dy)
    want = dy.double().sum(0)
    err = float((got.double() - want).norm() / want.norm())
    assert err <= 5.8 * 2 ** -24, err * 2 ** 24


def test_one_tensor_in_two_places_and_a_graph_run_twice():
    """Gate and up projection share weight and bias; the graph is kept."""
    x, ws, bs, dy = _make((50,), 64, 128, torch.bfloat16, True, "shared")
    _, _, dg, du, _, dbg, dbu, _ = _run(x, [ws[0], ws[0], ws[2]], [bs[0], bs[0], bs[2]], "gelu", None, dy)
    w, b = ws[0].detach().requires_grad_(True), bs[0].detach().requires_grad_(True)
    y = flash_gated_feed_forward(x, w, w, ws[2], b, b, bs[2], "gelu")
    for keep in (True, False):
        gw, gb = torch.autograd.grad(y, (w, b), dy, retain_graph=keep)
        assert torch.equal(gw, dg + du) and torch.equal(gb, dbg + dbu)


def test_activation_extremes():
    """Gates far into both tails: the activation and its derivative stay finite
    and right (a silu of -100 is -0, of 100 is 100)."""
    d = 8
    x = torch.eye(d, device=DEV)
    gates = torch.tensor([-200.0, -100.0, -20.0, -6.0, 6.0, 20.0, 100.0, 200.0], device=DEV)
    wg, wu, wd = torch.diag(gates), torch.eye(d, device=DEV), torch.eye(d, device=DEV)
    for act in ("silu", "gelu", "gelu_tanh"):
        got = _run(x, [wg, wu, wd], [None] * 3, act, None, torch.ones(d, d, device=DEV))
        want = ffn64(x, wg, wu, wd, None, None, None, act, valid_rows(x.shape, None), torch.ones(d, d, device=DEV))
        for name, a, b in zip(NAMES, got, want):
            if a is not None:
                # 1.5e-7 of the gate (gelu) and a few 2^-24 of the values
                assert float((a.detach().double() - b).abs().max()) <= 200 * 1.6e-7 + 1e-6 * float(b.abs().max()), (act, name)


def test_rows_do_not_touch_each_other():
    x, ws, bs, _ = _make((200,), 64, 128, torch.bfloat16, True, "rows")
    clean = flash_gated_feed_forward(x, *ws, *bs)
    y = x.clone()
    y[5], y[70], y[199, 3] = float("nan"), float("inf"), float("-inf")
    got = flash_gated_feed_forward(y, *ws, *bs)
    keep = [i for i in range(200) if i not in (5, 70, 199)]
    assert torch.equal(got[keep], clean[keep])
    assert bool(got[5].isnan().all()) and not bool(got[70].isfinite().any())


def test_features_that_end_inside_a_step_read_nothing_else():
    """D and F of no whole k step: the elements after a row's end (here NaN, in the
    rows' own storage) stay out of its sums."""
    x, ws, bs, dy = _make((100,), 40, 72, torch.bfloat16, True, "tail")
    wide = torch.full((100, 64), float("nan"), device=DEV, dtype=torch.bfloat16)
    gwide = wide.clone()
    wide[:, :40], gwide[:, :40] = x, dy
    a = _run(x, ws, bs, "silu", None, dy)
    b = _run(wide[:, :40], ws, bs, "silu", None, gwide[:, :40])
    for name, p, q in zip(NAMES, a, b):
        assert torch.equal(p, q), name


def test_gradient_against_differences():
    x, ws, bs, dy = _make((9,), 24, 40, torch.float32, True, "differences")
    tensors = [x, *ws, *bs]
    gen = torch.Generator().manual_seed(3)
    loss = lambda ts: float((flash_gated_feed_forward(*ts, "gelu").double() * dy.double()).sum())  # noqa: E731
    grads = _run(x, ws, bs, "gelu", None, dy)[1:]
    h = 2.0 ** -7
    for i, g in enumerate(grads):
        v = torch.randn(g.shape, generator=gen).to(DEV)
        at = lambda k: loss([t + k * h * v if j == i else t for j, t in enumerate(tensors)])  # noqa: E731
        # fourth-order difference: 216 outputs of order 1 off by about 1e-6 over 12 h, and h^4 terms
        got = (8 * (at(1) - at(-1)) - (at(2) - at(-2))) / (12 * h)
        want = float((g.double() * v.double()).sum())
        assert abs(got - want) <= 2e-3 * float(g.double().norm() * v.double().norm()), (i, got, want)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_bitwise_repeatable_and_on_another_stream(dtype):
    t = TYPES[dtype]
    lens = torch.randint(0, 301, (12,), generator=torch.Generator().manual_seed(1)).to(DEV)
    x, ws, bs, dy = _make((12, 300), 128, 264, t, True, (dtype, "repeat"))
    a = _run(x, ws, bs, "silu", lens, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = _run(x, ws, bs, "silu", lens, dy)
    side.synchronize()
    for name, p, q in zip(NAMES, a, b):
        assert torch.equal(p, q), name


def test_replays_in_a_graph():
    lens = torch.tensor([40, 3, 0, 17, 22, 40, 1, 9], device=DEV, dtype=torch.int32)
    x, ws, bs, dy = _make((8, 40), 96, 136, torch.bfloat16, True, "graph")

    def step():
        got = _run(x, ws, bs, "gelu", lens, dy)
        return [got[0].detach(), *got[1:]]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()
    for i in range(3):
        x.mul_(-1.25)
        lens.copy_(torch.roll(lens, 1))
        for t in static:
            t.fill_(float("nan"))
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for name, a, c in zip(NAMES, static, want):
            assert torch.equal(a, c), f"replay {i}: {name}"


def test_offsets_past_32_bits():
    """Hidden rows of more than 4 GiB (2^21 + 77 tokens of 1032), forward and
    gradients: the last tokens against the definition, the weights' gradients
    with only those tokens' dy nonzero."""
    rows, d, f, last = 2 ** 21 + 77, 32, 1032, 300
    x, ws, bs, _ = _make((last,), d, f, torch.bfloat16, True, "large")
    big = torch.zeros(rows, d, device=DEV, dtype=torch.bfloat16)
    big[-last:] = x
    dy = torch.zeros_like(big)
    dy[-last:] = torch.randn(last, d, generator=torch.Generator().manual_seed(2)).to(DEV, torch.bfloat16)
    got = _run(big, ws, bs, "silu", None, dy)
    want = ffn64(x, *ws, *bs, "silu", valid_rows(x.shape, None), dy[-last:])
    _compare([got[0][-last:], got[1][-last:], *got[2:]], want, torch.bfloat16)


def test_double_backward_and_stale_inputs_are_refused():
    x, ws, bs, dy = _make((5,), 16, 24, torch.float32, False, "twice")
    x.requires_grad_(True)
    g = torch.autograd.grad(flash_gated_feed_forward(x, *ws).sum(), x, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="twice"):
        g.sum().backward()
    for i in range(4):
        args = [t.detach().clone() for t in (x, *ws)]
        z = args[0].detach().requires_grad_(True) * 1.0
        y = flash_gated_feed_forward(z, *args[1:])
        with torch.no_grad():
            (z if i == 0 else args[i]).add_(1.0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward(dy)


@pytest.mark.parametrize("biases", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_host_extension_and_python_path_agree_bitwise(monkeypatch, dtype, biases):
    from flash_spacetime_amd import _lib

    assert _lib.host() is not None
    lens = torch.tensor([5, 0, 12], device=DEV)
    for key, lead, sl in (("rows", (33,), None), ("pad", (3, 12), lens), ("one", (), None)):
        x, ws, bs, dy = _make(lead, 40, 72, TYPES[dtype], biases, (dtype, key))
        a = _run(x, ws, bs, "gelu", sl, dy)
        with monkeypatch.context() as m:
            m.setattr(_lib, "host", lambda: None)
            c = _run(x, ws, bs, "gelu", sl, dy)
        for p, q in zip(a, c):
            assert (p is None) == (q is None) and (p is None or torch.equal(p, q))


def test_saved_tensor_hooks_see_what_the_backward_keeps():
    x, ws, bs, dy = _make((10,), 64, 96, torch.float32, True, "hooks")
    x.requires_grad_(True)
    seen = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: seen.append(tuple(t.shape)) or t.cpu(), lambda t: t.to(DEV)):
        y = flash_gated_feed_forward(x, *ws, *bs)
    assert (10, 64) in seen and seen.count((10, 96)) == 3  # x; the hidden rows and, in float32, both projections
    want = torch.autograd.grad(flash_gated_feed_forward(x, *ws, *bs), x, dy)[0]
    assert torch.equal(torch.autograd.grad(y, x, dy)[0], want)


def test_refusals():
    x, ws, bs, _ = _make((2, 3), 16, 24, torch.float32, True, "refusals")
    good = dict(x=x, w_gate=ws[0], w_up=ws[1], w_down=ws[2], b_gate=bs[0], b_up=bs[1], b_down=bs[2])
    bad = [
        (dict(x=x.double()), "bfloat16"), (dict(w_gate=ws[0].half()), "w_gate"), (dict(w_gate=ws[2]), "w_gate"),
        (dict(w_up=ws[1][:8]), "w_up"), (dict(w_down=ws[0]), "w_down"), (dict(b_gate=bs[2]), "b_gate"),
        (dict(b_up=bs[1].half()), "b_up"), (dict(b_down=bs[0]), "b_down"), (dict(activation="tanh"), "activation"),
        (dict(seqlens=torch.tensor([1], device=DEV)), "seqlens"), (dict(seqlens=torch.tensor([True, False], device=DEV)), "integer"),
        (dict(x=x[0], seqlens=torch.tensor([1, 2], device=DEV)), "padded"),
    ]
    for kwargs, what in bad:
        with pytest.raises(ValueError, match=what):
            flash_gated_feed_forward(**{**good, **kwargs})
    odd = torch.randn(4, 12, device=DEV)
    with pytest.raises(ValueError, match="multiples of 8"):
        flash_gated_feed_forward(odd, torch.randn(24, 12, device=DEV), torch.randn(24, 12, device=DEV), torch.randn(12, 24, device=DEV))
    with pytest.raises(RuntimeError, match="GPU"):
        flash_gated_feed_forward(**{**good, "w_up": ws[1].cpu()})


@pytest.mark.parametrize("name", ["fst_layer_norm_forward", "fst_layer_norm_backward", "fst_ffn_forward", "fst_ffn_backward"])
@pytest.mark.parametrize("status", [-1, -2, -3, -4])
def test_failed_calls_raise_and_refused_ones_take_the_python_path(name, status):
    """The library's entry points replaced by host functions that return a status
    (nothing is launched): a refused forward goes to the Python path, which runs
    it; any other failure is raised, once."""
    import ctypes

    from flash_spacetime_amd import _lib, flash_layer_norm

    base = ("fst_supported", "fst_forward_workspace_bytes", "fst_forward", "fst_backward_workspace_bytes", "fst_backward",
            "fst_last_error")
    block = ("fst_layer_norm_forward", "fst_layer_norm_backward_workspace_bytes", "fst_layer_norm_backward",
             "fst_ffn_forward", "fst_ffn_backward_workspace_bytes", "fst_ffn_backward")
    lib, calls = _lib.load(), []
    res, args = _lib.SIGNATURES[name]
    stub = ctypes.CFUNCTYPE(res, *args)(lambda *_: calls.append(name) or status)

    def bind(**stubs):
        _lib.host().bind_library(*(ctypes.cast(stubs.get(n, getattr(lib, n)), ctypes.c_void_p).value for n in base + block))

    x, ws, bs, dy = _make((6,), 16, 24, torch.float32, True, "stubs")

    def step():
        if "norm" not in name:
            return _run(x, ws, bs, "silu", None, dy)
        leaf = x.clone().requires_grad_(True)
        y = flash_layer_norm(leaf)
        return [y, *torch.autograd.grad(y, leaf, dy)]

    want = step()
    try:
        bind(**{name: stub})
        if status in (-1, -2) and name.endswith("forward"):
            assert all(torch.equal(a, b) for a, b in zip(step(), want))
        else:
            with pytest.raises(RuntimeError, match="flash_layer_norm" if "norm" in name else "flash_gated_feed_forward"):
                step()
    finally:
        bind()
    assert calls == [name]
    assert all(torch.equal(a, b) for a, b in zip(step(), want))
