"""CPU tests of the feed-forward's choice of tiles: every compiled tile is some
call's, and the query's refusals."""

import ctypes

import pytest

from flash_spacetime_amd import _lib

needs_lib = pytest.mark.skipif(not _lib.LIB_PATH.exists(), reason="libflash_spacetime.so not built")


def _tiles(dtype, rows, d, f):
    out = (ctypes.c_int32 * 6)()
    assert _lib.load().fst_ffn_tiles(dtype, 1, rows, d, f, out) == _lib.FST_OK
    return list(out)


@needs_lib
@pytest.mark.parametrize("dtype", [_lib.FST_BF16, _lib.FST_F16, _lib.FST_F32])
def test_every_tile_is_some_calls(dtype):
    """Gate, output, the projections' gradients, x's gradient, the weights' gradients:
    float32 has no 256-wide tile, 16-bit types no 64-wide one of the projections'
    gradients (that kernel is not compiled)."""
    seen = [set() for _ in range(5)]
    for rows in (1, 64, 65, 129, 300, 1000, 3000, 7640, 20000, 65536, 196608):
        for d in (8, 64, 136, 384, 520, 768, 1024):
            for f in (8, 72, 256, 392, 1024, 2752):
                for s, t in zip(seen, _tiles(dtype, rows, d, f)):
                    s.add(t)
    wide = set() if dtype == _lib.FST_F32 else {256}
    back = {16, 64, 128} if dtype == _lib.FST_F32 else {16, 128, 256}
    assert seen == [{16, 64, 128} | wide, {16, 64, 128} | wide, back, {16, 64, 128} | wide, {128} | wide]


@needs_lib
def test_runs_of_the_weights_gradients():
    """At least 256 rows a run where there is more than one, at most 64 runs."""
    for dtype in (_lib.FST_BF16, _lib.FST_F32):
        for rows in (0, 1, 255, 511, 512, 5000, 196608, 2 ** 31 - 1 - 65536):
            for d, f in ((8, 8), (384, 1024), (1024, 2752)):
                runs = _tiles(dtype, rows, d, f)[5]
                assert 1 <= runs <= 64 and (runs == 1 or runs * 256 <= rows)


@needs_lib
def test_tile_query_refusals():
    lib, out = _lib.load(), (ctypes.c_int32 * 6)()
    assert lib.fst_ffn_tiles(7, 1, 10, 16, 16, out) == _lib.FST_EINVAL and "dtype" in _lib.last_error()
    assert lib.fst_ffn_tiles(0, -1, 10, 16, 16, out) == _lib.FST_EINVAL and "negative" in _lib.last_error()
    assert lib.fst_ffn_tiles(0, 1, 10, 12, 16, out) == _lib.FST_EUNSUPPORTED and "multiples of 8" in _lib.last_error()
    assert lib.fst_ffn_tiles(0, 1, 2 ** 31 - 65536, 16, 16, out) == _lib.FST_EUNSUPPORTED and "rows" in _lib.last_error()
    assert lib.fst_ffn_tiles(0, 1, 10, 16, 16, None) == _lib.FST_EINVAL and "null" in _lib.last_error()
