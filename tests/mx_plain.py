"""Plain statements of the 4-bit block format and of the quantized key/value cache, in 64 bits on the
CPU: what the tests of those operators compare with."""

from __future__ import annotations

import math

import torch

BLOCK = 32
VALUES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def quant(x):
    """(codes 0..15 one a byte, scale bytes) of the blocks of x's last dimension."""
    v = x.detach().cpu().double().unflatten(-1, (-1, BLOCK))
    most = v.abs().amax(-1)
    finite = torch.isfinite(v).all(-1)
    safe = torch.where(finite, most, torch.ones_like(most))
    byte = (torch.frexp(safe).exponent - 1 - 2 + 127).clamp_min(0)  # frexp: most in [0.5, 1)
    byte = torch.where(safe == 0, 0, byte)
    q = torch.where(finite[..., None], v, torch.zeros_like(v)).abs() * torch.pow(
        2.0, 127.0 - byte.double())[..., None]
    # the nearest of the eight magnitudes, the even index where two are as near
    off = (q[..., None] - VALUES).abs()
    best = off.amin(-1, keepdim=True)
    near = off == best
    even = torch.arange(8) % 2 == 0
    code = torch.where((near & even).any(-1), (near & even).int().argmax(-1), near.int().argmax(-1))
    code = code + 8 * torch.signbit(v).int()
    code = torch.where(finite[..., None], code, torch.zeros_like(code))
    byte = torch.where(finite, byte, torch.full_like(byte, 255))
    return code.flatten(-2).to(torch.uint8), byte.to(torch.uint8)


def pack(code):
    c = code.unflatten(-1, (-1, 2)).int()
    return (c[..., 0] + 16 * c[..., 1]).to(torch.uint8)


def unpack(packed):
    p = packed.detach().cpu().view(torch.uint8).int()
    return torch.stack([p % 16, p // 16], -1).flatten(-2)


def values(code, byte):
    """The values of codes (one a byte) in binary64; NaN where the scale byte is 255."""
    code, byte = code.cpu().int(), byte.detach().cpu().view(torch.uint8).double()
    v = VALUES[code % 8] * torch.where(code >= 8, -1.0, 1.0)
    s = torch.where(byte == 255, math.nan, torch.pow(2.0, byte - 127))
    return (v.unflatten(-1, (-1, BLOCK)) * s[..., None]).flatten(-2)


def norm_rows(x, weight, eps, residual=None):
    """(y, after_res) of (residual add +) RMSNorm, each step rounded as the operators define it: the
    sum of squares in binary64, the row's scalar step by step to binary32, y at both of its products."""
    dtype = x.dtype
    a = x.cpu().float()
    if residual is not None:
        a = a + residual.cpu().float()
    total = a.double().square().sum(-1, keepdim=True).float()
    v = (total.double() / float(x.shape[-1])).float() + torch.tensor(eps, dtype=torch.float32)
    rho = (1.0 / v.double().sqrt().float().double()).float()
    y = ((a * rho).to(dtype).float() * weight.cpu().float()).to(dtype)
    return y, a.to(dtype)


def vector_codes(x, kind):
    """(codes, scales) of each vector along x's last dimension: int8 and fp8 codes in their own type
    with binary32 scales, 4-bit codes packed with scale bytes."""
    if kind == "mxfp4":
        code, byte = quant(x)
        return pack(code), byte
    v = x.detach().cpu().float()
    most = torch.nan_to_num(v.abs(), nan=0.0, posinf=math.inf).amax(-1)  # NaN is ignored
    if kind == "int8":
        scale = (most.double() / 127).float()
        inverse = (127 / most.double()).float()
        q = (v * inverse[..., None]).round().clamp(-127, 127)
        return torch.nan_to_num(q, nan=0.0).to(torch.int8), scale
    scale = (most.double() / 448).float().clamp_min(1.0 / (448.0 * 512.0))
    q = (v.double() / scale.double()[..., None]).float()
    q = torch.where(torch.isnan(q), torch.full_like(q, 448.0), q)
    return q.clamp(-448, 448).to(torch.float8_e4m3fn), scale


def vector_values(codes, scales, kind, dtype):
    """What the codes read back as: the product in binary32, rounded to dtype."""
    if kind == "mxfp4":
        return values(unpack(codes), scales).to(dtype)
    return (codes.cpu().float() * scales.cpu()[..., None]).to(dtype)


def same(a, b):
    """Bit equality, any NaN equal to any."""
    a, b = a.detach().cpu(), b.detach().cpu()
    if a.dtype != b.dtype or a.shape != b.shape:
        return False
    if not a.is_floating_point():
        return torch.equal(a, b)
    nan = torch.isnan(a.float()) & torch.isnan(b.float())
    ints = {1: torch.int8, 2: torch.int16, 4: torch.int32, 8: torch.int64}[a.element_size()]
    return bool(((a.contiguous().view(ints) == b.contiguous().view(ints)) | nan).all())
