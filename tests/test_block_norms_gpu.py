"""SpacetimeBlock with other modules in its norms' places, and as an earlier version pickled it."""

import copy

import pytest
import torch
from torch import nn

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from flash_spacetime_amd import SpacetimeBlock

DEV = "cuda"


class Norm(nn.Module):
    """A layer norm of another class: its parameters under the usual names."""

    def __init__(self, like):
        super().__init__()
        self.weight, self.bias, self.eps = like.weight, like.bias, like.eps


def _block():
    torch.manual_seed(3)
    block = SpacetimeBlock(64, 4, hidden=128, device=DEV)
    with torch.no_grad():
        for n in (block.norm1, block.norm2):
            n.weight.uniform_(0.5, 1.5)
            n.bias.normal_()
    return block, (torch.randn(2, 9, 64, device=DEV), torch.randn(2, 9, 5, device=DEV), torch.tensor([9, 4], device=DEV))


def test_a_layer_norm_of_another_class_stays_one():
    block, args = _block()
    want = block(*args)
    other = copy.deepcopy(block)
    other.norm1, other.norm2 = Norm(other.norm1), Norm(other.norm2)
    assert torch.equal(other(*args), want)


def test_a_block_of_an_earlier_version_runs():
    """Pickled before there were experts, it has no attributes for them."""
    block, args = _block()
    want = block(*args)
    old = copy.deepcopy(block)
    del old.__dict__["experts"], old.__dict__["top_k"]
    assert torch.equal(old(*args), want)
