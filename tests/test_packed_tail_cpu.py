"""CPU tests of fst_zero_tail's refusals (before any launch)."""

import pytest

from flash_spacetime_amd import _lib

needs_lib = pytest.mark.skipif(not _lib.LIB_PATH.exists(), reason="libflash_spacetime.so not built")


@needs_lib
def test_zero_tail_refusals():
    lib = _lib.load()
    call = lambda b=2, t=3, cu=16, rows=16, nbytes=32: lib.fst_zero_tail(b, t, cu, rows, nbytes, None)  # noqa: E731
    assert call(b=-1) == _lib.FST_EINVAL and call(t=-1) == _lib.FST_EINVAL and "negative" in _lib.last_error()
    assert call(cu=None) == _lib.FST_EINVAL and call(rows=None) == _lib.FST_EINVAL and "null" in _lib.last_error()
    assert call(nbytes=24) == _lib.FST_EINVAL and call(rows=8) == _lib.FST_EINVAL and "16" in _lib.last_error()
    assert call(t=2 ** 31 - 1, nbytes=2 ** 60) == _lib.FST_EINVAL and "2^63" in _lib.last_error()
    assert call(t=0, cu=None, rows=None) == _lib.FST_OK and call(nbytes=0, rows=None) == _lib.FST_OK
