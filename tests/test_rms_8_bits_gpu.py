"""flash_rms_norm_fp8's rounding: q = y / scale, rounded once, bit for bit.

The rows are ones and eps is 0, so that y is the weight itself. Scales of up to 18 bits are
exact (448 has three), and so are the weights that stand at a border between two 8-bit
values (five bits) times the scale. The quotient then stands on the border and goes to the even
neighbour; the product with the scale's rounded reciprocal does not.
"""

import pytest
import torch

from tests._block import TYPES
from tests._cases import seed_of

pytestmark = pytest.mark.gpu

if torch.cuda.is_available():
    from flash_spacetime_amd import flash_rms_norm_fp8

DEV = "cuda"


def _weights(n, gen):
    """(w, scale): float32 weights of both signs, the largest 448 scale."""
    scale = float(2 * int(torch.randint(1, 1 << 17, (1,), generator=gen)) + 1) * 2.0 ** -20
    border = 1 + (2 * torch.randint(0, 8, (n,), generator=gen) + 1) / 16  # between two values of three bits
    w = border * 2.0 ** torch.randint(-6, 8, (n,), generator=gen) * scale
    w[::3] = scale * torch.rand(len(w[::3]), generator=gen)  # and any others
    w *= torch.randint(0, 2, (n,), generator=gen) * 2 - 1
    w[n // 2] = 448 * scale
    return w, scale


@pytest.mark.parametrize("n", [64, 256, 1024, 8192])
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_8_bits_are_the_quotient_rounded_once(dtype, n):
    gen = torch.Generator().manual_seed(seed_of("8 bits", dtype, n))
    for offset in (0, 1):  # rows on 16 bytes, and off them
        x = torch.ones(3, n + 8, device=DEV, dtype=TYPES[dtype])[:, offset:n + offset]
        for _ in range(8):
            w, scale = _weights(n, gen)
            q, got = flash_rms_norm_fp8(x, w.to(DEV), 0.0)
            assert got.tolist() == [scale] * 3
            want = (w / torch.tensor(scale)).to(torch.float8_e4m3fn).view(torch.uint8)
            assert torch.equal(q.view(torch.uint8).cpu(), want.expand(3, n))


def test_8_bits_of_infinite_weights():
    """Beside an infinite value the others' quotients are 0; its own is not a number."""
    w = torch.ones(64, device=DEV)
    w[5], w[9] = float("inf"), -2.0
    q, scale = flash_rms_norm_fp8(torch.ones(2, 64, device=DEV), w, 0.0)
    assert bool(scale.isinf().all()) and bool(q.float()[:, 5].isnan().all())
    assert bool((q.float()[:, torch.arange(64) != 5] == 0).all())
