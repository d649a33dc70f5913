"""The tiled forms of the product of 4-bit operands on the GPU, each at sizes that reach it."""

import pytest
import torch

import mcoplib_amd._C  # noqa: F401
from gpu_util import DEV, say
from test_gpu_mxfp4_mm import _operand, _product, _values

pytestmark = pytest.mark.gpu


# fp32 outputs are turned through the LDS that the first of the tiles in turn lies in, and without a bias
# no second barrier comes between: sizes whose last tile along K (256 each) is in that place, which is
# every other one with two in turn and every third with three.
LAST_IN_FIRST_PLACE = [
    (1024, 4096, 4096),  # 128 x 128, three in turn, 16 tiles
    (700, 4099, 4096),   # the same past both ends
    (2048, 4096, 1280),  # 128 x 128, two in turn, 5 tiles
    (2048, 4096, 4352),  # the same, 17 tiles
    (1500, 4096, 4096),  # 192 x 128, three in turn, 16 tiles
    (900, 4099, 4096),
    (2048, 4099, 2304),  # 256 x 256, two in turn, 9 tiles
    (4096, 4096, 2304),
]


@pytest.mark.parametrize("M,N,K", LAST_IN_FIRST_PLACE)
def test_outputs_over_the_last_tile(M, N, K):
    """Exact sums (test_gpu_mxfp4_mm.py), so that one operand read from what is already an output shows."""
    say(f"mxfp4 mm over the last tile {M}x{N}x{K}")
    a, b = _operand(M, K, M + K), _operand(N, K, N + 3 * K)
    ref = (_values(a).to(DEV) @ _values(b).to(DEV).t()).float()
    for _ in range(3):
        got = _product(a, b)
        assert torch.equal(got, ref), int((got != ref).sum())
