"""4-bit blocks on the GPU: codes and scales bit for bit against a plain statement in 64 bits, over
every type, ragged widths, strides and alignments, and special values; the norm-quant operator against
the norm's rows rounded step by step; what the operators must leave alone."""

import math

import pytest
import torch

import mcoplib_amd._C  # noqa: F401
import mx_plain
from gpu_util import DEV, randn, say, weight
from mcoplib import custom_ops

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _check_quant(x, what):
    code, byte = mx_plain.quant(x)
    got, scale = custom_ops.mxfp4_quant(x)
    assert mx_plain.same(got, mx_plain.pack(code)), what
    assert mx_plain.same(scale, byte), what
    back = custom_ops.mxfp4_dequant(got, scale, x.dtype)
    assert mx_plain.same(back, mx_plain.values(code, byte).to(x.dtype)), what


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,H", [(1, 32), (1, 64), (3, 96), (5, 4128), (257, 160), (1000, 1056),
                                 (2, 65536), (4097, 32), (64, 5120)])
def test_quant_and_back(T, H, dtype):
    say(f"mxfp4 quant {T}x{H} {dtype}")
    x = randn((T, H), T * 7 + H, dtype, scale=3.0)
    x[:, ::17] *= 50  # outliers: blocks with most values at the smallest codes
    _check_quant(x.to(DEV), "random")


@pytest.mark.parametrize("dtype", TYPES)
def test_every_magnitude(dtype):
    """Every 16-bit pattern (for fp32: every such upper half), finite or not, in blocks of its own kind
    and beside a value 2^k times as large: ties, subnormals, both zeros, infinities, NaN."""
    say(f"mxfp4 every magnitude {dtype}")
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16)
    v = bits.view(torch.float16 if dtype == torch.float16 else torch.bfloat16)
    x = v.float().to(dtype) if dtype == torch.float32 else v
    _check_quant(x.reshape(-1, 4096).to(DEV), "all patterns in order")
    finite = x[torch.isfinite(x)]
    few = finite[torch.randperm(finite.numel(), generator=torch.Generator().manual_seed(1))]
    few = few[:63488 // 31 * 31].reshape(-1, 31)
    for k in (0, 1, 2, 3, 4):
        most = (few.abs().amax(-1, keepdim=True).float() * 2.0 ** k).to(dtype)
        _check_quant(torch.cat([few, most], -1).to(DEV), f"2^{k}")


@pytest.mark.parametrize("dtype", TYPES)
def test_special_blocks(dtype):
    say(f"mxfp4 special blocks {dtype}")
    tiny = torch.finfo(dtype).smallest_normal
    rows = torch.zeros(12, 96, dtype=dtype)
    rows[1, 40] = math.inf
    rows[2, 95] = math.nan
    rows[3, :32] = -0.0
    rows[4, 3] = torch.finfo(dtype).max
    rows[5, 64] = -torch.finfo(dtype).max
    rows[6] = tiny
    rows[7] = tiny * torch.arange(96) / 16  # subnormals, and zero
    rows[8, 32:64] = -math.inf
    rows[9] = torch.arange(96) % 13 - 6.0
    rows[10] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 4.0]).repeat(12)  # ties
    rows[11] = -rows[10]
    _check_quant(rows.to(DEV), "special")


@pytest.mark.parametrize("dtype", TYPES)
def test_strided_and_misaligned_rows(dtype):
    say(f"mxfp4 strides {dtype}")
    flat = randn((1, 40000), 5, dtype).to(DEV)[0]
    for offset in (0, 1, 3, 8):
        for stride in (96, 97, 128, 131):
            _check_quant(flat.as_strided((37, 96), (stride, 1), offset), (offset, stride))
    _check_quant(flat.as_strided((3, 5, 64), (5 * 70, 70, 1), 2), "3-D")
    _check_quant(flat[:64].expand(4, 64), "rows of one memory")
    codes, scale = custom_ops.mxfp4_quant(flat[:1024].view(8, 128))
    out = torch.full((1 + 8 * 128 + 7,), 9.0, dtype=dtype, device=DEV)
    torch.ops._C.mxfp4_dequant(out[1:1025].view(8, 128), codes, scale)  # misaligned output
    assert mx_plain.same(out[1:1025].view(8, 128),
                         mx_plain.values(mx_plain.unpack(codes), scale).to(dtype))
    assert out[0] == 9 and bool((out[1025:] == 9).all())


@pytest.mark.parametrize("dtype", TYPES)
def test_every_code_and_scale_reads_back(dtype):
    say(f"mxfp4 dequant {dtype}")
    code = torch.arange(32, dtype=torch.uint8).remainder(16).repeat(256, 1)
    byte = torch.arange(256, dtype=torch.int32).to(torch.uint8)[:, None]
    got = custom_ops.mxfp4_dequant(mx_plain.pack(code).to(DEV), byte.to(DEV), dtype)
    assert mx_plain.same(got, mx_plain.values(code, byte).to(dtype))


def test_other_code_types_and_untouched_memory():
    x = randn((3, 64), 2, torch.bfloat16).to(DEV)
    code, byte = mx_plain.quant(x)
    buf = torch.full((4 + 3 * 32 + 4,), 77, dtype=torch.uint8, device=DEV)
    sbuf = torch.full((1 + 6 + 3,), 77, dtype=torch.uint8, device=DEV)
    torch.ops._C.mxfp4_quant(buf[4:100].view(3, 32).view(torch.float4_e2m1fn_x2), x,
                             sbuf[1:7].view(3, 2).view(torch.float8_e8m0fnu))
    assert mx_plain.same(buf[4:100].view(3, 32), mx_plain.pack(code))
    assert mx_plain.same(sbuf[1:7].view(3, 2), byte)
    assert bool((buf[:4] == 77).all() and (buf[100:] == 77).all())
    assert sbuf[0] == 77 and bool((sbuf[7:] == 77).all())
    empty = custom_ops.mxfp4_quant(x[:0])
    assert empty[0].shape == (0, 32) and empty[1].shape == (0, 2)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,H", [(1, 32), (3, 96), (1, 5120), (64, 4096), (300, 1056), (7, 8192),
                                 (2, 16416), (3, 32768), (2, 40960), (1, 131072)])
@pytest.mark.parametrize("residual", [False, True])
def test_norm_quant(T, H, residual, dtype):
    say(f"rms_norm_mxfp4_quant {T}x{H} {dtype} residual={residual}")
    x, w = randn((T, H), H + T, dtype, scale=2.0), weight(H, 3, dtype)
    r = randn((T, H), 9, dtype) if residual else None
    y, after = mx_plain.norm_rows(x, w, 1e-6, r)
    code, byte = mx_plain.quant(y)
    got, scale, a = custom_ops.rms_norm_mxfp4_quant(x.to(DEV), w.to(DEV), 1e-6,
                                                    r.to(DEV) if residual else None)
    assert mx_plain.same(got, mx_plain.pack(code)) and mx_plain.same(scale, byte)
    assert (a is None) if not residual else mx_plain.same(a, after)


@pytest.mark.parametrize("H", [96, 5120, 65568])
@pytest.mark.parametrize("into", ["residual", "input", "misaligned"])
def test_norm_quant_in_place_and_misaligned(H, into):
    """after_res in the residual's or the input's own memory; tensors one element off alignment."""
    say(f"rms_norm_mxfp4_quant H={H} {into}")
    dtype, T = torch.bfloat16, 5
    x, r, w = randn((T, H), 1, dtype), randn((T, H), 2, dtype), weight(H, 3, dtype)
    y, after = mx_plain.norm_rows(x, w, 1e-5, r)
    code, byte = mx_plain.quant(y)
    move = lambda t: t.to(DEV)  # noqa: E731
    if into == "misaligned":
        move = lambda t: torch.cat([t.flatten()[:1], t.flatten()]).to(DEV)[1:].view(t.shape)  # noqa: E731
    xd, rd, wd = move(x), move(r), move(w)
    got = torch.empty(T, H // 2, dtype=torch.uint8, device=DEV)
    scale = torch.empty(T, H // 32, dtype=torch.uint8, device=DEV)
    target = xd if into == "input" else rd
    torch.ops._C.rms_norm_mxfp4_quant(got, xd, wd, scale, 1e-5, rd, target)
    assert mx_plain.same(got, mx_plain.pack(code)) and mx_plain.same(scale, byte)
    assert mx_plain.same(target, after)
    assert mx_plain.same(xd if into != "input" else rd, x if into != "input" else r)


def test_norm_quant_of_special_rows():
    """A NaN makes its row NaN, an infinity too (inf * 0); a zero row is zero codes of scale 0; a NaN
    weight spoils its own blocks alone."""
    dtype, H = torch.bfloat16, 128
    x, w = randn((5, H), 1, dtype), weight(H, 2, dtype)
    x[1, 7], x[2, 7], x[3] = math.nan, math.inf, 0.0
    w2 = w.clone()
    w2[40] = math.nan
    for ww in (w, w2):
        y, _ = mx_plain.norm_rows(x, ww, 1e-6)
        code, byte = mx_plain.quant(y)
        got, scale, _ = custom_ops.rms_norm_mxfp4_quant(x.to(DEV), ww.to(DEV), 1e-6)
        assert mx_plain.same(got, mx_plain.pack(code)) and mx_plain.same(scale, byte)


def test_large_rows_pass_32_bit_offsets():
    """More than 2^31 elements: the last rows of the tensor, and the first of its second launch."""
    T, H = (1 << 20) + 3, 2080
    say(f"mxfp4 quant of {T * H} elements")
    x = torch.zeros(T, H, dtype=torch.bfloat16, device=DEV)
    tail = randn((3, H), 4, torch.bfloat16)
    x[-3:] = tail.to(DEV)
    x[516222:516225] = tail.to(DEV)
    codes, scale = custom_ops.mxfp4_quant(x)
    code, byte = mx_plain.quant(tail)
    for rows in (slice(T - 3, T), slice(516222, 516225)):
        assert mx_plain.same(codes[rows], mx_plain.pack(code)) and mx_plain.same(scale[rows], byte)
    assert int(codes[:1000].sum()) == 0 and int(codes[600000:700000].sum()) == 0
    del x
    back = custom_ops.mxfp4_dequant(codes, scale, torch.bfloat16)
    assert mx_plain.same(back[-3:], mx_plain.values(code, byte).to(torch.bfloat16))
