"""CPU tests of the RMS norm and mixture-of-experts operators' host side: refusals of
the Python operators and of the C entry points (before any launch), workspace queries,
tiles, and the block's parameters."""

import ctypes

import pytest
import torch

from flash_spacetime_amd import (ExpertOrder, SpacetimeBlock, _lib, flash_expert_combine, flash_expert_dispatch,
                                 flash_expert_feed_forward, flash_expert_route, flash_expert_sort, flash_rms_norm,
                                 flash_rms_norm_fp8)

needs_lib = pytest.mark.skipif(not _lib.LIB_PATH.exists(), reason="libflash_spacetime.so not built")


def test_there_is_no_cpu_path():
    x, ids = torch.randn(4, 16), torch.zeros(4, 2, dtype=torch.int32)
    order = ExpertOrder(ids[:, 0], ids, torch.zeros(3, dtype=torch.int32))
    for call in (lambda: flash_rms_norm(x), lambda: flash_rms_norm_fp8(x), lambda: flash_expert_route(x, 2),
                 lambda: flash_expert_sort(ids, 2), lambda: flash_expert_dispatch(x, order),
                 lambda: flash_expert_combine(x, x[:, :2], order),
                 lambda: flash_expert_feed_forward(x, ids[0], x[None], x[None], x[None])):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def test_8_bits_ask_for_no_gradient():
    with pytest.raises(ValueError, match="no derivative"):
        flash_rms_norm_fp8(torch.randn(4, 16, requires_grad=True))


@needs_lib
def test_rms_norm_refusals():
    lib = _lib.load()
    for name in ("fst_rms_norm_forward", "fst_rms_norm_fp8"):
        f = getattr(lib, name)
        last = 16 if name.endswith("fp8") else None  # scales are needed, rstd is not

        def fwd(dt=0, pt=1, b=2, l=3, n=8, xs=8, eps=1e-5, x=16, y=16, r=None, s=None, rs=0, scale=last):
            tail = (scale, s) if name.endswith("fp8") else (s, scale)
            return f(dt, pt, b, l, n, x, xs, r, rs, None, None, eps, y, *tail, None)

        assert fwd(dt=7) == _lib.FST_EINVAL and "dtype" in _lib.last_error()
        assert fwd(pt=2) == _lib.FST_EINVAL and "param_dtype" in _lib.last_error()
        assert fwd(b=-1) == _lib.FST_EINVAL and "negative" in _lib.last_error()
        assert fwd(n=0) == _lib.FST_EINVAL and "feature" in _lib.last_error()
        assert fwd(n=16385, xs=16385) == _lib.FST_EUNSUPPORTED and "16384" in _lib.last_error()
        assert fwd(b=65536, l=65536) == _lib.FST_EUNSUPPORTED and "rows" in _lib.last_error()
        assert fwd(xs=7) == _lib.FST_EINVAL and "stride" in _lib.last_error()
        assert fwd(r=16, rs=7, s=16) == _lib.FST_EINVAL and "stride" in _lib.last_error()
        assert fwd(x=None) == _lib.FST_EINVAL and fwd(y=None) == _lib.FST_EINVAL and "null" in _lib.last_error()
        assert fwd(r=16, rs=8) == _lib.FST_EINVAL and "null" in _lib.last_error()
        assert fwd(eps=-1.0) == _lib.FST_EINVAL and fwd(eps=float("nan")) == _lib.FST_EINVAL and "eps" in _lib.last_error()
        assert fwd(b=0) == _lib.FST_OK
        if last:
            assert fwd(scale=None) == _lib.FST_EINVAL and "null" in _lib.last_error()
    bwd = lambda ws, nbytes, dy=16, dw=16, dx=16, dys=8: lib.fst_rms_norm_backward(  # noqa: E731
        0, 1, 2, 3, 8, 16, 8, None, None, 16, dy, dys, None, 0, dx, dw, ws, nbytes, None)
    assert lib.fst_rms_norm_backward_workspace_bytes(0, 2, 3, 8) > 0
    assert lib.fst_rms_norm_backward_workspace_bytes(0, 2, 3, 0) == 0
    assert bwd(16, 1) == _lib.FST_EWORKSPACE and "workspace" in _lib.last_error()
    assert bwd(None, 0, dy=None) == _lib.FST_EINVAL and "null" in _lib.last_error()
    assert bwd(None, 0, dys=5) == _lib.FST_EINVAL and "stride" in _lib.last_error()
    assert bwd(None, 0, dw=None, dx=None) == _lib.FST_OK  # nothing is asked for


@needs_lib
def test_route_and_sort_refusals():
    lib = _lib.load()

    def route(dt=1, b=2, l=3, e=8, k=2, logits=16, stride=8, w=16, ids=16):
        return lib.fst_expert_route(dt, b, l, e, k, 1, logits, stride, None, w, ids, None)

    assert route(dt=3) == _lib.FST_EINVAL and "dtype" in _lib.last_error()
    assert route(l=-1) == _lib.FST_EINVAL and "negative" in _lib.last_error()
    for e, k in ((0, 1), (8, 0), (8, 9)):
        assert route(e=e, k=k) == _lib.FST_EINVAL and "top_k" in _lib.last_error()
    assert route(e=513, stride=513) == _lib.FST_EUNSUPPORTED and route(e=20, k=17, stride=20) == _lib.FST_EUNSUPPORTED
    assert route(b=65536, l=32767) == _lib.FST_EUNSUPPORTED and "slots" in _lib.last_error()
    assert route(stride=7) == _lib.FST_EINVAL and "stride" in _lib.last_error()
    for null in ("logits", "w", "ids"):
        assert route(**{null: None}) == _lib.FST_EINVAL and "null" in _lib.last_error()
    assert route(b=0, logits=None) == _lib.FST_OK

    def back(normalize=1, logits=None, stride=8, dw=16, dl=16):
        return lib.fst_expert_route_backward(1, 2, 3, 8, 2, normalize, logits, stride, None, 16, 16, dw, dl, None)

    assert back(0) == _lib.FST_EINVAL and back(dw=None) == _lib.FST_EINVAL and back(dl=None) == _lib.FST_EINVAL
    assert back(0, 16, 7) == _lib.FST_EINVAL and "stride" in _lib.last_error()

    def sort(slots=10000, e=8, ids=16, offsets=16, ws=16, nbytes=1 << 30):
        return lib.fst_expert_sort(slots, e, ids, 16, 16, offsets, ws, nbytes, None)

    assert sort(slots=-1) == _lib.FST_EINVAL and "negative" in _lib.last_error()
    assert sort(e=0) == _lib.FST_EINVAL and sort(e=513) == _lib.FST_EUNSUPPORTED
    assert sort(slots=0x7FFFFFFF) == _lib.FST_EUNSUPPORTED and "slots" in _lib.last_error()
    assert sort(ids=None) == _lib.FST_EINVAL and sort(offsets=None) == _lib.FST_EINVAL and "null" in _lib.last_error()
    need = lib.fst_expert_sort_workspace_bytes(10000, 8)
    assert need > 0 and lib.fst_expert_sort_workspace_bytes(100, 8) == 0 and lib.fst_expert_sort_workspace_bytes(1, 0) == 0
    assert sort(nbytes=need - 1) == _lib.FST_EWORKSPACE and sort(ws=None) == _lib.FST_EWORKSPACE


@needs_lib
def test_every_sort_has_its_counts_in_reach():
    """A workgroup adds up the counts of all: at most 32 loads a thread (csrc/fst_experts.hip)."""
    lib = _lib.load()
    for e in (1, 2, 7, 8, 63, 64, 100, 127, 128, 255, 256, 511, 512):
        for slots in (8193, 20000, 524288, 524289, 10 ** 7, 0x7FFFFFFF - 65536):
            blocks = lib.fst_expert_sort_workspace_bytes(slots, e) // (4 * (e + 1))
            width = 1 << e.bit_length()
            assert 1 <= blocks <= 32 * max(1024 // width, 1) + 64, (e, slots, blocks)


@needs_lib
def test_mover_refusals():
    lib = _lib.load()

    def spread(dt=0, wt=1, tokens=5, k=2, n=8, rows=10, x=16, xs=8, place=16, used=16, w=None, back=None, bs=0, out=16, dw=None):
        return lib.fst_expert_spread(dt, wt, tokens, k, n, rows, x, xs, place, used, w, back, bs, out, dw, None)

    def gather(dt=0, wt=1, tokens=5, k=2, n=8, rows=10, x=16, xs=8, place=16, out=16):
        return lib.fst_expert_gather(dt, wt, tokens, k, n, rows, x, xs, place, None, out, None)

    for f in (spread, gather):
        assert f(dt=9) == _lib.FST_EINVAL and "dtype" in _lib.last_error()
        assert f(wt=2) == _lib.FST_EINVAL and "weight_dtype" in _lib.last_error()
        assert f(tokens=-1) == _lib.FST_EINVAL and f(rows=-1) == _lib.FST_EINVAL and "negative" in _lib.last_error()
        assert f(k=0) == _lib.FST_EINVAL and f(n=0, xs=0) == _lib.FST_EINVAL
        assert f(k=17) == _lib.FST_EUNSUPPORTED and f(n=16385, xs=16385) == _lib.FST_EUNSUPPORTED
        assert f(rows=1 << 31) == _lib.FST_EUNSUPPORTED and f(tokens=1 << 30) == _lib.FST_EUNSUPPORTED
        assert f(xs=7) == _lib.FST_EINVAL and "stride" in _lib.last_error()
        assert f(x=None) == _lib.FST_EINVAL and f(place=None) == _lib.FST_EINVAL and "null" in _lib.last_error()
    assert spread(used=None) == _lib.FST_EINVAL and spread(back=16, bs=8) == _lib.FST_EINVAL
    assert spread(back=16, bs=7, dw=16) == _lib.FST_EINVAL and "stride" in _lib.last_error()
    assert spread(out=None) == _lib.FST_OK and spread(tokens=0, rows=0) == _lib.FST_OK and gather(tokens=0) == _lib.FST_OK
    assert gather(out=None) == _lib.FST_EINVAL


@needs_lib
def test_expert_feed_forward_refusals():
    lib = _lib.load()

    def fwd(dt=0, act=0, rows=6, e=2, d=16, f=32, x=16, xs=16, offsets=16, wg=16, gate=None, up=None, y=16):
        return lib.fst_expert_ffn_forward(dt, act, rows, e, d, f, x, xs, offsets, wg, 16, 16, 16, gate, up, y, None)

    assert fwd(dt=5) == _lib.FST_EINVAL and "dtype" in _lib.last_error()
    assert fwd(act=3) == _lib.FST_EINVAL and "activation" in _lib.last_error()
    assert fwd(rows=-1) == _lib.FST_EINVAL and "negative" in _lib.last_error()
    assert fwd(e=0) == _lib.FST_EINVAL and "expert" in _lib.last_error()
    assert fwd(e=513) == _lib.FST_EUNSUPPORTED and "experts" in _lib.last_error()
    for d, f in ((12, 32), (16, 36), (0, 8), (8, 4)):
        assert fwd(d=d, f=f, xs=d + 16) == _lib.FST_EUNSUPPORTED and "multiples of 8" in _lib.last_error()
    assert fwd(d=32768, f=8192, xs=32768) == _lib.FST_EUNSUPPORTED and fwd(rows=0x7FFFFFFF) == _lib.FST_EUNSUPPORTED
    assert fwd(xs=8) == _lib.FST_EINVAL and fwd(xs=20) == _lib.FST_EINVAL and fwd(xs=1 << 31) == _lib.FST_EINVAL
    assert fwd(x=8) == _lib.FST_EINVAL and "16 bytes" in _lib.last_error()
    assert fwd(wg=None) == _lib.FST_EINVAL and fwd(offsets=None) == _lib.FST_EINVAL and "null" in _lib.last_error()
    assert fwd(gate=16, up=16) == _lib.FST_EINVAL and "float32" in _lib.last_error()
    assert fwd(dt=1, gate=16) == _lib.FST_EINVAL
    assert fwd(rows=0) == _lib.FST_OK

    def bwd(ws=16, nbytes=1 << 40, dy=16, dys=16, dx=16, dw=16, dt=0, offsets=16):
        return lib.fst_expert_ffn_backward(dt, 0, 6, 2, 16, 32, 16, 16, offsets, 16, 16, 16, 16, None, None, dy, dys, dx, dw,
                                           None, None, ws, nbytes, None)

    assert bwd(dy=None) == _lib.FST_EINVAL and bwd(offsets=None) == _lib.FST_EINVAL and "null" in _lib.last_error()
    assert bwd(dt=1) == _lib.FST_EINVAL  # float32 needs gate and up
    assert bwd(dys=12) == _lib.FST_EINVAL and "stride" in _lib.last_error()
    assert bwd(dx=8) == _lib.FST_EINVAL and "16 bytes" in _lib.last_error()
    need = lib.fst_expert_ffn_backward_workspace_bytes(0, 6, 2, 16, 32)
    assert need > 0 and lib.fst_expert_ffn_backward_workspace_bytes(0, 6, 0, 16, 32) == 0
    assert bwd(nbytes=need - 1) == _lib.FST_EWORKSPACE and bwd(ws=None) == _lib.FST_EWORKSPACE
    assert bwd(dx=None, dw=None) == _lib.FST_OK


@needs_lib
def test_tiles_follow_the_runs():
    """Few rows of each expert take small tiles, however many there are in all."""
    lib, tiles = _lib.load(), (ctypes.c_int32 * 6)()
    of = lambda *a: (lib.fst_expert_ffn_tiles(*a, tiles), list(tiles))[1]  # noqa: E731
    assert of(0, 16, 8, 768, 2048)[:4] == [16] * 4
    assert of(0, 65536, 32, 1024, 1376)[0] == 256 and of(0, 65536, 32, 1024, 1376)[5] == 1
    assert of(0, 4096, 512, 256, 256)[1] == 64 and of(1, 16384, 8, 512, 704)[0] == 128
    assert lib.fst_expert_ffn_tiles(0, 16, 0, 64, 64, tiles) == _lib.FST_EINVAL


def test_block_with_experts_has_their_parameters():
    blk = SpacetimeBlock(96, 4, norm="rms", experts=6, top_k=3, hidden=128)
    names = {n: tuple(p.shape) for n, p in blk.named_parameters()}
    assert names["router.weight"] == (6, 96) and names["experts_gate"] == names["experts_up"] == (6, 128, 96)
    assert names["experts_down"] == (6, 96, 128) and names["norm1.weight"] == (96,)
    assert not any(n.startswith("ffn_") or n in ("norm1.bias", "norm2.bias", "router.bias") for n in names)
    assert float(blk.experts_down.detach().abs().max()) <= 128 ** -0.5
    plain = SpacetimeBlock(96, 4)
    assert not any("experts" in n or "router" in n for n, _ in plain.named_parameters())
    with pytest.raises(ValueError, match="norm"):
        SpacetimeBlock(96, 4, norm="batch")
    with pytest.raises(ValueError, match="top_k"):
        SpacetimeBlock(96, 4, experts=2, top_k=3)
