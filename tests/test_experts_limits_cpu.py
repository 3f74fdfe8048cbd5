"""CPU tests of the mixture of experts' limits: what is past them is refused by the call,
or the module, that is asked for it, before any launch."""

import pytest

from flash_spacetime_amd import SpacetimeBlock


@pytest.mark.parametrize("experts,top_k,what", [(513, 2, "512"), (40, 17, "16"), (0, 1, "top_k"), (4, 0, "top_k")])
def test_block_refuses_what_its_router_does(experts, top_k, what):
    with pytest.raises(ValueError, match=what):
        SpacetimeBlock(32, 4, hidden=64, experts=experts, top_k=top_k)


def test_block_takes_the_router_s_most():
    block = SpacetimeBlock(32, 4, hidden=8, experts=512, top_k=16)
    assert (block.experts, block.top_k, block.router.weight.shape[0]) == (512, 16, 512)
