"""CPU tests of the layer norm and feed-forward operators' host side: refusals of
the Python operators and of the C entry points (before any launch), workspace
queries, the rows the kernels are given, and the binding against the header."""

import re
from pathlib import Path

import pytest
import torch

from flash_spacetime_amd import _lib, flash_gated_feed_forward, flash_layer_norm
from flash_spacetime_amd.norm import batch_of_rows, token_rows

HEADER = Path(__file__).resolve().parents[1] / "include" / "flash_spacetime.h"
needs_lib = pytest.mark.skipif(not _lib.LIB_PATH.exists(), reason="libflash_spacetime.so not built")


def test_there_is_no_cpu_path():
    x = torch.randn(4, 16)
    with pytest.raises(RuntimeError, match="GPU"):
        flash_layer_norm(x)
    with pytest.raises(RuntimeError, match="GPU"):
        flash_gated_feed_forward(x, x, x, x)


def test_binding_has_the_headers_arguments():
    text = re.sub(r"/\*.*?\*/", "", HEADER.read_text(), flags=re.S)
    for name in _lib.SIGNATURES:
        m = re.search(rf"\b{name}\s*\(([^)]*)\)", text)
        args = [a for a in m.group(1).split(",") if a.strip() not in ("", "void")]
        kinds = _lib.SIGNATURES[name][1]
        assert len(args) == len(kinds), name
        for a, k in zip(args, kinds):
            want = ("P" if "*" in a else "l" if "int64_t" in a else "L" if "size_t" in a else "f" if "float" in a else "i")
            if k is not None and hasattr(k, "_type_") and isinstance(k._type_, str):
                assert k._type_ == want, (name, a)


@needs_lib
def test_norm_refusals():
    lib = _lib.load()
    fwd = lambda dt=0, pt=1, b=2, l=3, n=8, xs=8, eps=1e-5, x=16, y=16, r=None, s=None, rs=0: lib.fst_layer_norm_forward(  # noqa: E731
        dt, pt, b, l, n, x, xs, r, rs, None, None, None, eps, y, s, None, None)
    assert fwd(dt=7) == _lib.FST_EINVAL and "dtype" in _lib.last_error()
    assert fwd(pt=2) == _lib.FST_EINVAL and "param_dtype" in _lib.last_error()
    assert fwd(b=-1) == _lib.FST_EINVAL and "negative" in _lib.last_error()
    assert fwd(n=0) == _lib.FST_EINVAL and "feature" in _lib.last_error()
    assert fwd(n=16385, xs=16385) == _lib.FST_EUNSUPPORTED and "16384" in _lib.last_error()
    assert fwd(b=65536, l=65536) == _lib.FST_EUNSUPPORTED and "rows" in _lib.last_error()
    assert fwd(xs=7) == _lib.FST_EINVAL and "stride" in _lib.last_error()
    assert fwd(x=None) == _lib.FST_EINVAL and "null" in _lib.last_error()
    assert fwd(r=16, rs=8) == _lib.FST_EINVAL and "null" in _lib.last_error()
    assert fwd(eps=-1.0) == _lib.FST_EINVAL and fwd(eps=float("nan")) == _lib.FST_EINVAL and "eps" in _lib.last_error()
    assert fwd(b=0) == _lib.FST_OK
    bwd = lambda ws, nbytes, dy=16, dw=16, dx=16: lib.fst_layer_norm_backward(  # noqa: E731
        0, 1, 2, 3, 8, 16, 8, None, None, 16, dy, 8, None, 0, dx, dw, None, ws, nbytes, None)
    assert lib.fst_layer_norm_backward_workspace_bytes(0, 2, 3, 8) > 0
    assert lib.fst_layer_norm_backward_workspace_bytes(0, 2, 3, 0) == 0
    assert bwd(16, 1) == _lib.FST_EWORKSPACE and "workspace" in _lib.last_error()
    assert bwd(None, 0, dy=None) == _lib.FST_EINVAL and "null" in _lib.last_error()
    assert bwd(None, 0, dw=None, dx=None) == _lib.FST_OK  # nothing is asked for


@needs_lib
def test_feed_forward_refusals():
    lib = _lib.load()

    def fwd(dt=0, act=0, b=2, l=3, d=16, f=32, x=16, xs=16, wg=16, lens=None, gate=None, up=None, y=16, rowmap=None):
        return lib.fst_ffn_forward(dt, act, b, l, d, f, x, xs, wg, 16, 16, None, None, None, lens, 16, gate, up, rowmap,
                                   y, None)

    assert fwd(dt=5) == _lib.FST_EINVAL and "dtype" in _lib.last_error()
    assert fwd(act=3) == _lib.FST_EINVAL and "activation" in _lib.last_error()
    assert fwd(l=-1) == _lib.FST_EINVAL and "negative" in _lib.last_error()
    for d, f in ((12, 32), (16, 36), (0, 8), (8, 4)):
        assert fwd(d=d, f=f, xs=d + 16) == _lib.FST_EUNSUPPORTED and "multiples of 8" in _lib.last_error()
    assert fwd(d=65544, xs=65544) == _lib.FST_EUNSUPPORTED
    assert fwd(d=32768, f=8192, xs=32768) == _lib.FST_EUNSUPPORTED and "elements" in _lib.last_error()
    assert fwd(b=65536, l=32768) == _lib.FST_EUNSUPPORTED and "rows" in _lib.last_error()
    assert fwd(xs=8) == _lib.FST_EINVAL and "stride" in _lib.last_error()
    assert fwd(xs=1 << 31) == _lib.FST_EINVAL and "stride" in _lib.last_error()
    assert fwd(xs=20) == _lib.FST_EINVAL and "stride" in _lib.last_error()
    assert fwd(x=8) == _lib.FST_EINVAL and "16 bytes" in _lib.last_error()
    assert fwd(wg=None) == _lib.FST_EINVAL and "null" in _lib.last_error()
    assert fwd(gate=16, up=16) == _lib.FST_EINVAL and "float32" in _lib.last_error()
    assert fwd(dt=1, gate=16) == _lib.FST_EINVAL and fwd(lens=16) == _lib.FST_EINVAL and "null" in _lib.last_error()
    assert fwd(b=0) == _lib.FST_OK

    def bwd(ws=16, nbytes=1 << 40, dy=16, dys=16, dx=16, dw=16, dt=0):
        return lib.fst_ffn_backward(dt, 0, 2, 3, 16, 32, 16, 16, 16, 16, 16, None, None, None, 16, None, None, None, dy, dys,
                                    dx, dw, None, None, None, None, None, ws, nbytes, None)

    assert bwd(dy=None) == _lib.FST_EINVAL and "null" in _lib.last_error()
    assert bwd(dt=1) == _lib.FST_EINVAL and "null" in _lib.last_error()  # float32 needs gate and up
    assert bwd(dys=12) == _lib.FST_EINVAL and "stride" in _lib.last_error()
    assert bwd(dx=8) == _lib.FST_EINVAL and "16 bytes" in _lib.last_error()
    need = lib.fst_ffn_backward_workspace_bytes(0, 2, 3, 16, 32)
    assert need > 0 and lib.fst_ffn_backward_workspace_bytes(0, 2, 3, 12, 32) == 0
    assert bwd(nbytes=need - 1) == _lib.FST_EWORKSPACE and bwd(ws=None) == _lib.FST_EWORKSPACE
    assert bwd(dx=None, dw=None) == _lib.FST_OK


def test_rows_are_taken_in_place_where_they_can_be():
    x = torch.arange(600.0).view(10, 60)
    assert token_rows(x) == (x, 60)
    view = x[:, 20:40]
    got, stride = token_rows(view)
    assert got is view and stride == 60
    assert token_rows(x.view(2, 5, 60)[:, :, :30])[1] == 60
    for odd in (x.t(), x[:, ::2], x[:1].expand(10, 60), x.view(2, 5, 60)[:, :3]):
        got, stride = token_rows(odd)
        assert got.is_contiguous() and stride == odd.shape[-1] and torch.equal(got, odd)
    got, stride = token_rows(x[:, 1:33], 16)
    assert got.is_contiguous() and got.data_ptr() % 16 == 0 and torch.equal(got, x[:, 1:33])
    assert token_rows(x[3], 16)[1] == 60 and token_rows(x[0:0], 16)[1] == 60
    one = x[2:3].expand(1, 60)
    assert token_rows(one)[1] == 60


def test_lengths_are_checked():
    x = torch.zeros(3, 7, 8)
    assert batch_of_rows(x, None) == (1, 21, None)
    b, length, lens = batch_of_rows(x, torch.tensor([1, 2, 3]))
    assert (b, length) == (3, 7) and lens.dtype == torch.int32
    for bad in (torch.tensor([1, 2]), torch.tensor([[1, 2, 3]]), torch.tensor([1.0, 2, 3]), torch.tensor([True, True, False])):
        with pytest.raises(ValueError, match="seqlens"):
            batch_of_rows(x, bad)
    with pytest.raises(ValueError, match="padded"):
        batch_of_rows(x[0], torch.tensor([1, 2, 3]))
