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


class Rms(nn.Module):
    """A root-mean-square norm of another class: it has no bias."""

    def __init__(self, like):
        super().__init__()
        self.weight, self.eps = like.weight, like.eps


def _block(norm="layer"):
    torch.manual_seed(3)
    block = SpacetimeBlock(64, 4, hidden=128, device=DEV, norm=norm)
    with torch.no_grad():
        for n in (block.norm1, block.norm2):
            n.weight.uniform_(0.5, 1.5)
            if norm == "layer":
                n.bias.normal_()
    return block, (torch.randn(2, 9, 64, device=DEV), torch.randn(2, 9, 5, device=DEV), torch.tensor([9, 4], device=DEV))


@pytest.mark.parametrize("norm,cls", [("layer", Norm), ("rms", Rms)])
def test_norms_of_another_class_stay_what_they_are(norm, cls):
    block, args = _block(norm)
    want = block(*args)
    other = copy.deepcopy(block)
    other.norm1, other.norm2 = cls(other.norm1), cls(other.norm2)
    assert torch.equal(other(*args), want)


def test_a_block_of_an_earlier_version_runs():
    """Pickled before there were experts, it has no attributes for them."""
    block, args = _block()
    want = block(*args)
    old = copy.deepcopy(block)
    del old.__dict__["experts"], old.__dict__["top_k"]
    assert torch.equal(old(*args), want)
