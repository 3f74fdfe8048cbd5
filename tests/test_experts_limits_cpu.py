"""CPU tests of the mixture of experts' limits: what is past them is refused by the call,
or the module, that is asked for it, before any launch."""

import pytest

from flash_spacetime_amd import SpacetimeBlock, _lib
from tests.test_expert_tiles_gpu import CASES, tiles

needs_lib = pytest.mark.skipif(not _lib.LIB_PATH.exists(), reason="libflash_spacetime.so not built")


@pytest.mark.parametrize("experts,top_k,what", [(513, 2, "512"), (40, 17, "16"), (0, 1, "top_k"), (4, 0, "top_k")])
def test_block_refuses_what_its_router_does(experts, top_k, what):
    with pytest.raises(ValueError, match=what):
        SpacetimeBlock(32, 4, hidden=64, experts=experts, top_k=top_k)


def test_block_takes_the_router_s_most():
    block = SpacetimeBlock(32, 4, hidden=8, experts=512, top_k=16)
    assert (block.experts, block.top_k, block.router.weight.shape[0]) == (512, 16, 512)


@needs_lib
def test_movers_of_an_order_refuse():
    lib = _lib.load()

    def spread(tokens=5, k=2, rows=10, xs=8, place=16, order=16, order_rows=10, used=16, out=16):
        return lib.fst_expert_spread_order(0, 1, tokens, k, 8, rows, 16, xs, place, order, order_rows, used, None, None, 0, out,
                                           None, None)

    def gather(tokens=5, k=2, rows=10, xs=8, place=16, used=16, out=16):
        return lib.fst_expert_gather_order(0, 1, tokens, k, 8, rows, 16, xs, place, used, None, out, None)

    for f in (spread, gather):
        assert f(tokens=-1) == _lib.FST_EINVAL and f(rows=-1) == _lib.FST_EINVAL and "negative" in _lib.last_error()
        assert f(k=17) == _lib.FST_EUNSUPPORTED and f(rows=1 << 31) == _lib.FST_EUNSUPPORTED
        assert f(xs=7) == _lib.FST_EINVAL and "stride" in _lib.last_error()
        assert f(place=None) == _lib.FST_EINVAL and "null" in _lib.last_error()
    assert spread(order_rows=-1) == _lib.FST_EINVAL and "order" in _lib.last_error()
    assert spread(used=None) == _lib.FST_EINVAL and gather(out=None) == _lib.FST_EINVAL
    assert spread(out=None) == _lib.FST_OK and spread(tokens=0, rows=0) == _lib.FST_OK and gather(tokens=0) == _lib.FST_OK


@needs_lib
@pytest.mark.parametrize("k", [2, 4, 8, 16])
def test_products_of_sizes_past_64_bits(k):
    """Tokens times slots that come out small, or below 0, in 64 bits."""
    lib = _lib.load()
    for tokens in (2 ** 64 // k - 2 ** 33, 2 ** 62 // k, 2 ** 63 // k, 2 ** 63 - 1):
        tokens = min(tokens, 2 ** 63 - 1)
        assert lib.fst_expert_gather(0, 1, tokens, k, 8, 10, 16, 8, 16, None, 16, None) == _lib.FST_EUNSUPPORTED
        assert lib.fst_expert_spread(0, 1, tokens, k, 8, 10, 16, 8, 16, 16, None, None, 0, 16, None, None) == _lib.FST_EUNSUPPORTED
    most = 2 ** 31 - 1
    for b, l in ((most, most), (most, 2 ** 30), (2 ** 30, most // k)):
        assert lib.fst_expert_route(1, b, l, 16, k, 1, 16, 16, None, 16, 16, None) == _lib.FST_EUNSUPPORTED, (b, l)
        assert lib.fst_expert_route_backward(1, b, l, 16, k, 1, None, 16, None, 16, 16, 16, 16, None) == _lib.FST_EUNSUPPORTED


@needs_lib
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_every_tile_of_the_experts_products_is_a_tested_cases(dtype):
    """Gate, output, the projections' gradients, x's gradient, the weights' gradients written
    directly and in pieces: the cases of test_expert_tiles_gpu.py reach what is compiled."""
    of = [tiles(dtype, *c[:4]) for c in CASES]
    assert of == [c[5 if dtype == "f32" else 4] for c in CASES]
    wide = set() if dtype == "f32" else {256}
    back = {16, 64, 128} if dtype == "f32" else {16, 128, 256}
    assert [{t[i] for t in of} for i in range(4)] == [{16, 64, 128} | wide, {16, 64, 128} | wide, back, {16, 64, 128} | wide]
    assert {(t[4], t[5] > 1) for t in of} >= {(e, s) for e in {128} | wide for s in (False, True)}


@needs_lib
def test_every_sort_s_counts_are_all_added_up():
    """A workgroup adds up the counts of all, at most 32 loads a thread; the workspace's
    rounding to 256 bytes holds at most 63 // (e + 1) workgroups' counts more."""
    lib = _lib.load()
    for e in range(1, 513):
        for slots in (8193, 20000, 524288, 524289, 10 ** 7, 0x7FFFFFFF - 65536):
            blocks = lib.fst_expert_sort_workspace_bytes(slots, e) // (4 * (e + 1)) - 63 // (e + 1)
            assert blocks <= 32 * max(1024 // (1 << e.bit_length()), 1), (e, slots, blocks)
