"""Product of 4-bit operands on the GPU.

Two kinds of operands.  `exact`: scales of 1 and 2, so that every product is a multiple of 1/4 and
every partial sum below 2^24 quarters (6 * 6 * 4 * K * 4 < 2^24 for K <= 29127): binary32 holds each of
them, so the result is the same in any order and fp32 outputs are compared bit for bit.  `wide`: scales
over 2^-8..2^8, compared in 64 bits: each of the K additions is off by at most one step (2^-23) of a
partial sum, which is at most sum|a b|, and the output's rounding by half a step of its own type."""

import math

import pytest
import torch

import mcoplib_amd._C  # noqa: F401
import mx_plain
from gpu_util import DEV, say
from mcoplib import custom_ops

pytestmark = pytest.mark.gpu


def _operand(rows, K, seed, low=127, high=129):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (rows, K // 2), generator=g, dtype=torch.int32).to(torch.uint8)
    scale = torch.randint(low, high, (rows, K // 32), generator=g, dtype=torch.int32)
    return codes, scale.to(torch.uint8)


def _values(op):
    return mx_plain.values(mx_plain.unpack(op[0]), op[1])


def _fenced(t, before=64, fill=255):
    """t on the device between bytes that would spoil a result that read them (NaN scales)."""
    flat = t.contiguous().view(torch.uint8).flatten()
    buf = torch.full((before + flat.numel() + 512,), fill, dtype=torch.uint8, device=DEV)
    buf[before:before + flat.numel()] = flat.to(DEV)
    return buf[before:before + flat.numel()].view(t.shape)


def _product(a, b, dtype=torch.float32, bias=None, shift=0):
    """The operator's result, written between untouched elements; `shift` moves scales off dwords."""
    M, N = a[0].shape[0], b[0].shape[0]
    buf = torch.full((16 + M * N + 64,), 7.0, dtype=dtype, device=DEV)
    out = buf[16:16 + M * N].view(M, N)
    torch.ops._C.mxfp4_scaled_mm(out, _fenced(a[0]), _fenced(a[1], 64 + shift), _fenced(b[0]),
                                 _fenced(b[1], 64 + shift), bias)
    assert bool((buf[:16] == 7).all()) and bool((buf[16 + M * N:] == 7).all())
    return out


SHAPES = [(1, 1, 32), (1, 5, 64), (2, 16, 96), (3, 31, 160), (15, 128, 512), (16, 17, 544),
          (17, 257, 1056), (33, 64, 2048), (64, 130, 4096), (65, 96, 1120), (100, 100, 8192),
          (128, 129, 288), (200, 1000, 640), (256, 256, 1024), (257, 513, 1504), (512, 300, 2592),
          (1025, 260, 256)]


@pytest.mark.parametrize("M,N,K", SHAPES)
def test_exact_sums(M, N, K):
    say(f"mxfp4 mm exact {M}x{N}x{K}")
    a, b = _operand(M, K, M + K), _operand(N, K, N + 3 * K)
    ref = (_values(a) @ _values(b).t()).float()
    for shift in (0, 1):
        assert mx_plain.same(_product(a, b, shift=shift), ref), shift


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("M,N,K", [(1, 48, 5120), (7, 100, 1056), (40, 64, 4096), (130, 72, 2080),
                                   (300, 520, 3200), (64, 4099, 544)])
def test_wide_scales_bias_and_types(M, N, K, dtype):
    say(f"mxfp4 mm {M}x{N}x{K} {dtype}")
    a, b = _operand(M, K, 1, 119, 128), _operand(N, K, 2, 119, 128)
    va, vb = _values(a), _values(b)
    bias = torch.randn(N, generator=torch.Generator().manual_seed(3)).to(dtype)
    ref = va @ vb.t() + bias.double()
    got = _product(a, b, dtype, bias.to(DEV)).cpu().double()
    room = K * 2.0 ** -23 * (va.abs() @ vb.abs().t() + bias.double().abs())
    room = room + torch.finfo(dtype).eps / 2 * (ref.abs() + room) + 2.0 ** -25  # fp16 subnormals
    assert bool(((got - ref).abs() <= room).all()), float(((got - ref).abs() / room).max())


def test_extreme_scales():
    """Scales whose product leaves binary32's normal range, and zero codes under any scale."""
    a, b = _operand(4, 64, 1), _operand(4, 64, 2)
    a[1].fill_(250), b[1].fill_(4)  # 2^123 and 2^-123: the product is in range
    ref = (_values(a) @ _values(b).t()).float()
    assert mx_plain.same(_product(a, b), ref)
    a[0].zero_()
    assert bool((_product(a, b) == 0).all())
    a[1].fill_(0), b[1].fill_(254)
    assert bool((_product(a, b) == 0).all())


@pytest.mark.parametrize("M,N,K", [(5, 40, 96), (150, 140, 1056)])
def test_nan_scales_spoil_their_row_or_column(M, N, K):
    a, b = _operand(M, K, 1), _operand(N, K, 2)
    a[1][2, 1], b[1][7, K // 32 - 1] = 255, 255
    a[0][2], b[0][7] = 0x22, 0x22  # also where the codes are 1
    got = _product(a, b).cpu()
    nan = torch.zeros(M, N, dtype=torch.bool)
    nan[2], nan[:, 7] = True, True
    ref = (_values(a) @ _values(b).t()).float()
    assert torch.equal(torch.isnan(got), nan)
    assert mx_plain.same(got, torch.where(nan, torch.tensor(math.nan), ref))


def test_shapes_of_the_functional_form():
    a, b = _operand(6, 64, 1), _operand(10, 64, 2)
    a3 = (a[0].view(2, 3, 32).to(DEV), a[1].view(2, 3, 2).to(DEV))
    out = custom_ops.mxfp4_scaled_mm(*a3, b[0].to(DEV), b[1].to(DEV), torch.float32)
    assert out.shape == (2, 3, 10)
    assert mx_plain.same(out.view(6, 10), (_values(a) @ _values(b).t()).float())
    none = custom_ops.mxfp4_scaled_mm(a3[0][:0], a3[1][:0], b[0].to(DEV), b[1].to(DEV),
                                      torch.bfloat16)
    assert none.shape == (0, 3, 10)
    four = custom_ops.mxfp4_scaled_mm(
        a3[0].view(torch.float4_e2m1fn_x2), a3[1].view(torch.float8_e8m0fnu), b[0].to(DEV),
        b[1].to(DEV), torch.float32)
    assert torch.equal(four, out)
    with pytest.raises(RuntimeError, match="aligned to 16"):
        flat = torch.zeros(8 + 6 * 32, dtype=torch.uint8, device=DEV)
        custom_ops.mxfp4_scaled_mm(flat[8:].view(6, 32), a[1].to(DEV), b[0].to(DEV), b[1].to(DEV),
                                   torch.float32)


def test_random_shapes():
    """48 seeded shapes over the operator's range, bit for bit."""
    g = torch.Generator().manual_seed(11)
    u = torch.rand(48, 3, generator=g).tolist()
    for i, (x, y, z) in enumerate(u):
        M, N, K = int(1500 ** x), int(1500 ** y), 32 * int(256 ** z)
        say(f"mxfp4 mm random {i}: {M}x{N}x{K}")
        a, b = _operand(M, K, i), _operand(N, K, 100 + i)
        ref = (_values(a) @ _values(b).t()).float()
        assert mx_plain.same(_product(a, b, shift=i % 2), ref), (M, N, K)


# Sizes of every tile shape, each with rows and columns inside a tile and tails of K of one block, or none;
# with scales off dwords, which go through registers (test_gpu_mxfp4_mm_forms.py has every form by name).
LARGE = [(16, 8192, 8224), (3, 2050, 9248), (33, 4099, 8224), (40, 16400, 4128), (100, 8192, 5152),
         (100, 4099, 2080), (130, 2050, 4128), (700, 4099, 1056), (1030, 2050, 1568),
         (700, 4099, 5152), (900, 4099, 4128), (2300, 1700, 512), (2300, 1700, 544),
         (2100, 2050, 2080), (1300, 4099, 1056), (2500, 2500, 544), (2100, 4100, 3104),
         (3000, 3001, 1056), (4000, 4001, 544), (4096, 4096, 512), (500, 16300, 160),
         (500, 16300, 288), (500, 16300, 544), (1237, 4099, 5152), (1500, 3001, 4128),
         (250, 16300, 672), (250, 16300, 800), (250, 16300, 768), (700, 4099, 5248),
         (900, 4099, 4224), (250, 8100, 5152), (256, 8192, 5120), (400, 4099, 4224),
         (64, 16300, 128), (64, 16300, 384), (500, 4000, 640), (500, 4000, 2176)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,N,K", LARGE)
def test_exact_sums_of_large_products(M, N, K, dtype):
    """As test_exact_sums; the rounding to bf16 of an exact sum is one too.  The 64-bit product is
    made on the device."""
    say(f"mxfp4 mm large {M}x{N}x{K} {dtype}")
    a, b = _operand(M, K, M + K), _operand(N, K, N + 3 * K)
    ref = (_values(a).to(DEV) @ _values(b).to(DEV).t()).to(torch.float32).to(dtype)
    got = _product(a, b, dtype, shift=3)
    assert torch.equal(got, ref), int((got != ref).sum())
    bias = torch.randint(-8, 9, (N,), generator=torch.Generator().manual_seed(5)).to(dtype)
    ref = (_values(a).to(DEV) @ _values(b).to(DEV).t() + bias.to(DEV).double()).float().to(dtype)
    assert torch.equal(_product(a, b, dtype, bias.to(DEV)), ref)


@pytest.mark.parametrize("M,N,K", [(70, 4099, 2080), (900, 4099, 4128), (2100, 4100, 3104)])
def test_nan_scales_in_large_products(M, N, K):
    a, b = _operand(M, K, 1), _operand(N, K, 2)
    rows, columns = [0, 31, M - 1], [5, 64, N - 1]
    a[1][rows, K // 32 - 1], b[1][columns, 3] = 255, 255
    a[0][rows], b[0][columns] = 0x22, 0x22
    nan = torch.zeros(M, N, dtype=torch.bool)
    nan[rows], nan[:, columns] = True, True
    assert torch.equal(torch.isnan(_product(a, b)).cpu(), nan)


def test_operands_past_32_bit_offsets():
    """Weights of 8 GiB of codes: the columns at their end are those of the end alone (exact sums, so
    that the forms of the two products do not matter)."""
    N, K = (1 << 20) + 3, 16384
    g = torch.Generator(device=DEV).manual_seed(4)
    b = torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8, device=DEV)
    sb = torch.randint(127, 129, (N, K // 32), generator=g, dtype=torch.uint8, device=DEV)
    for M in (1, 40):
        say(f"mxfp4 mm {M}x{N}x{K}")
        a, sa = (t.to(DEV) for t in _operand(M, K, M))
        out = torch.empty(M, N, dtype=torch.float32, device=DEV)
        torch.ops._C.mxfp4_scaled_mm(out, a, sa, b, sb, None)
        for part in (slice(0, 70), slice(N - 131, N)):
            ref = (_values((a, sa)) @ _values((b[part], sb[part])).t()).float()
            assert mx_plain.same(out[:, part], ref)
