"""GPU tests of layer norm rows that end inside a 16-byte piece."""

import pytest
import torch

from tests._block import TYPES, norm64, valid_rows
from tests._cases import seed_of

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from flash_spacetime_amd import flash_layer_norm

DEV = "cuda"


@pytest.mark.parametrize("n", [1, 5, 47, 393, 1003])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_parameters_gradients_alone_of_rows_that_end_inside_a_piece(dtype, n):
    """Without x's gradient the backward writes no rows, and rows a multiple of 16
    bytes apart are aligned whatever their length: it has to read their last piece as
    one that ends inside. The rows stand in wider ones filled up with NaN, the last
    ending with its storage; the gradients have the bits of the call that
    forms x's gradient too (of rows stored one after another) and are the
    definition's: sums of 21 rows, a few 2^-24 of the terms beside the rounding to
    the parameters' type."""
    t = TYPES[dtype]
    gen = torch.Generator().manual_seed(seed_of("edges", dtype, n))
    wide = -(-n // 8) * 8 + 8

    def rows():
        store = torch.full((20 * wide + n,), float("nan"), device=DEV, dtype=t)
        view = store.as_strided((21, n), (wide, 1))
        view.copy_(torch.randn(21, n, generator=gen))
        assert view.data_ptr() % 16 == 0 and view.stride(0) * view.element_size() % 16 == 0
        return view

    x, dy = rows(), rows()
    params = [torch.randn(n, generator=gen).to(DEV).requires_grad_(True) for _ in range(2)]
    alone = torch.autograd.grad(flash_layer_norm(x, *params), params, dy)
    leaf = x.contiguous().requires_grad_(True)
    full = torch.autograd.grad(flash_layer_norm(leaf, *params), [leaf, *params], dy.contiguous())
    want = norm64(x, None, *params, 1e-5, valid_rows(x.shape, None), dy)[3:]
    for got, same, ref in zip(alone, full[1:], want):
        assert torch.equal(got, same)
        assert float((got.double().cpu() - ref).abs().max()) <= 256 * 2.0 ** -24 * 21 * (1 + n ** 0.5)
