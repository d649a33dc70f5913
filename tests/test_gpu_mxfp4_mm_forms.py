"""The tiled forms of the product of 4-bit operands on the GPU, each at sizes that reach it."""

import math

import pytest
import torch

import mcoplib_amd._C  # noqa: F401
import mx_plain
from gpu_util import DEV, say
from mcoplib_amd import _lib
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


# A size of each form, with rows and columns past a tile's end where the form is met at such.  Where
# scales go to LDS directly K is past 8 tiles, so that both places of scales are filled and read again, and
# a tile and a half past them or whole.
FORMS = [
    ((15, 500, 1056), "rows"),
    ((48, 2050, 2176), "32x32 by eight waves"),
    ((33, 4099, 2208), "32x32"),
    ((100, 4099, 8224), "64x64 by waves apart"),
    ((2300, 1700, 672), "64x64"),
    ((400, 4099, 4224), "64x64, three tiles, direct scales"),
    ((64, 16300, 2304), "64x64, three tiles, direct scales"),
    ((400, 4099, 4192), "64x64, three tiles"),
    ((250, 8100, 3200), "128x64, three tiles, direct scales"),
    ((256, 8192, 4096), "128x64, three tiles, direct scales"),
    ((250, 8100, 3232), "128x64, three tiles"),
    ((700, 4099, 5248), "128x128, three tiles, direct scales"),
    ((1024, 4096, 2304), "128x128, three tiles, direct scales"),
    ((700, 4099, 5280), "128x128, three tiles"),
    ((1300, 4099, 1184), "128x128"),
    ((1500, 3001, 2176), "192x128, three tiles, direct scales"),
    ((1500, 4096, 2304), "192x128, three tiles, direct scales"),
    ((1500, 3001, 2208), "192x128, three tiles"),
    ((2100, 4100, 2208), "256x256"),
]
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _on_device(op):
    """An operand's values in 64 bits on the device, its rows a part at a time."""
    parts = max(1, op[0].numel() >> 24)
    return torch.cat([_values(part).to(DEV) for part in zip(op[0].chunk(parts), op[1].chunk(parts))])


def _case(size, form, *scales):
    M, N, K = size
    assert _lib.mxfp4_mm_form(M, N, K) == form
    say(f"mxfp4 mm form {M}x{N}x{K}: {form}")
    return _operand(M, K, M + K, *scales), _operand(N, K, N + 3 * K, *scales)


@pytest.mark.parametrize("size,form", FORMS)
def test_exact_sums_of_every_form(size, form):
    """Each type, with a bias and without, aligned scales (and, where that is another way, unaligned):
    exact sums in 64 bits, rounded once."""
    a, b = _case(size, form)
    ref = _on_device(a) @ _on_device(b).t()
    bias = torch.randint(-8, 9, (size[1],), generator=torch.Generator().manual_seed(5)).to(DEV)
    for dtype in TYPES:
        for shift in (0, 3) if "direct" in form else (0,):
            got = _product(a, b, dtype, shift=shift)
            assert torch.equal(got, ref.float().to(dtype)), (dtype, shift)
            got = _product(a, b, dtype, bias.to(dtype), shift)
            assert torch.equal(got, (ref + bias).float().to(dtype)), (dtype, shift, "bias")


@pytest.mark.parametrize("size,form", FORMS)
def test_wide_scales_in_every_form(size, form):
    """Scales of 2^-8 to 1, a bias and each type, within what K additions of a step each (2^-23 of at most
    sum|a b|) and one rounding allow, as in test_gpu_mxfp4_mm.py."""
    a, b = _case(size, form, 119, 128)
    va, vb = _on_device(a), _on_device(b)
    ref, most = va @ vb.t(), va.abs() @ vb.abs().t()
    g = torch.Generator().manual_seed(3)
    bias = torch.randn(size[1], generator=g).to(DEV)
    for dtype in TYPES:
        add = bias.to(dtype)
        want = ref + add.double()
        off = (_product(a, b, dtype, add).double() - want).abs()
        room = size[2] * 2.0 ** -23 * (most + add.double().abs())
        room = room + torch.finfo(dtype).eps / 2 * (want.abs() + room) + 2.0 ** -25  # fp16 subnormals
        assert bool((off <= room).all()), (dtype, float((off / room).max()))


@pytest.mark.parametrize("size,form", FORMS)
def test_far_scales_in_every_form(size, form):
    """Scales of 2^-123 to 2^123 that cancel between the operands block by block: the sums stay exact, and
    a scale that is taken from another block is off by a power of two or far out of range."""
    a, b = _case(size, form)
    g = torch.Generator().manual_seed(9)
    e = torch.randint(4, 251, (size[2] // 32,), generator=g, dtype=torch.int32)
    plain = _on_device(a) @ _on_device(b).t()
    a = (a[0], (a[1].int() - 127 + e).to(torch.uint8))
    b = (b[0], (b[1].int() - 127 + 254 - e).to(torch.uint8))
    for shift in (0, 3) if "direct" in form else (0,):
        got = _product(a, b, shift=shift)
        assert torch.equal(got, plain.float()), shift


@pytest.mark.parametrize("size,form", FORMS)
def test_nan_scales_in_every_form(size, form):
    """A NaN scale in the first, an inner and the last block of a row or column, each in a row of its own:
    NaN there and nowhere else."""
    (M, N, K), blocks = size, size[2] // 32
    a, b = _case(size, form)
    ref = (_on_device(a) @ _on_device(b).t()).float()
    rows, columns = [0, M // 2, M - 1], [5, N // 2 + 1, N - 1]
    a[1][rows, [0, blocks - 1, blocks // 2]] = 255
    b[1][columns, [blocks - 1, blocks // 2 + 1, 0]] = 255
    ref[rows], ref[:, columns] = math.nan, math.nan
    for shift in (0, 3) if "direct" in form else (0,):
        assert mx_plain.same(_product(a, b, shift=shift), ref), shift
