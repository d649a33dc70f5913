"""Without a GPU: the 4-bit operators' and the quantized cache's schemas and Meta kernels, and what
their surfaces and the C ABI refuse before anything reaches a device."""

import ctypes

import pytest
import torch

import mcoplib._C  # noqa: F401
import mx_plain
from mcoplib import custom_ops
from mcoplib_amd import _C, _lib

BF = torch.bfloat16


def _u8(*shape):
    return torch.zeros(*shape, dtype=torch.uint8)


def test_schemas_name_their_outputs():
    writes = {"mxfp4_quant": ["result", "scale"], "mxfp4_dequant": ["result"],
              "rms_norm_mxfp4_quant": ["result", "scale", "after_res"],
              "mxfp4_scaled_mm": ["result"],
              "kv_cache_write_quant": ["key_cache", "value_cache", "key_scale", "value_scale"],
              "kv_cache_read_dequant": ["key", "value"]}
    for name, outs in writes.items():
        schema = getattr(torch.ops._C, name).default._schema
        assert [a.name for a in schema.arguments
                if a.alias_info is not None and a.alias_info.is_write] == outs, name
        assert not schema.returns


def test_meta_kernels_accept_meta_tensors():
    m = torch.device("meta")
    e = lambda *s, dtype=torch.uint8: torch.empty(*s, dtype=dtype, device=m)  # noqa: E731
    x = e(4, 64, dtype=BF)
    torch.ops._C.mxfp4_quant(e(4, 32), x, e(4, 2))
    torch.ops._C.mxfp4_dequant(x, e(4, 32), e(4, 2))
    torch.ops._C.rms_norm_mxfp4_quant(e(4, 32), x, e(64, dtype=BF), e(4, 2), 1e-6, x, x)
    torch.ops._C.mxfp4_scaled_mm(e(4, 8, dtype=BF), e(4, 32), e(4, 2), e(8, 32), e(8, 2), None)
    kv = e(4, 2, 64, dtype=BF)
    cache, scale = e(3, 16, 2, 64, dtype=torch.int8), e(3, 16, 2, dtype=torch.float32)
    torch.ops._C.kv_cache_write_quant(kv, kv, cache, cache, scale, scale,
                                      e(4, dtype=torch.int64))
    torch.ops._C.kv_cache_read_dequant(kv, kv, cache, cache, scale, scale,
                                       e(1, 3, dtype=torch.int32), e(2, dtype=torch.int32), None)


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 64, dtype=BF)
    with pytest.raises(RuntimeError, match="CUDA"):
        custom_ops.mxfp4_quant(x)
    with pytest.raises(RuntimeError, match="CUDA"):
        custom_ops.rms_norm_mxfp4_quant(x, torch.ones(64, dtype=BF), 1e-6, x)
    with pytest.raises(RuntimeError, match="CUDA"):
        custom_ops.mxfp4_scaled_mm(_u8(4, 32), _u8(4, 2), _u8(8, 32), _u8(8, 2), BF)
    with pytest.raises(NotImplementedError):
        torch.ops._C.mxfp4_quant(_u8(4, 32), x, _u8(4, 2))


@pytest.mark.parametrize("call,match", [
    (lambda x: _C.mxfp4_quant(_u8(4, 32), x.int(), _u8(4, 2)), "not implemented for 'Int'"),
    (lambda x: _C.mxfp4_quant(_u8(4, 24), x[:, :48], _u8(4, 1)), "multiple of the block of 32"),
    (lambda x: _C.mxfp4_quant(_u8(4, 31), x, _u8(4, 2)), "expected 4 rows of 32"),
    (lambda x: _C.mxfp4_quant(_u8(4, 32), x, _u8(4, 1)), "expected 4 rows of 2"),
    (lambda x: _C.mxfp4_quant(_u8(4, 32).int(), x, _u8(4, 2)), "uint8 or float4_e2m1fn_x2"),
    (lambda x: _C.mxfp4_quant(_u8(4, 32), x, torch.zeros(4, 2)), "uint8 or float8_e8m0fnu"),
    (lambda x: _C.mxfp4_quant(_u8(4, 64)[:, ::2], x, _u8(4, 2)), "result must be contiguous"),
    (lambda x: _C.mxfp4_quant(_u8(64, 2), x.t(), _u8(64, 1)), "last dimension of input"),
    (lambda x: _C.mxfp4_quant(_u8(2, 2, 2, 16), torch.zeros(2, 5, 2, 32)[:, :2], _u8(2, 2, 2, 1)),
     "uniformly strided"),
    (lambda x: _C.mxfp4_dequant(x.int(), _u8(4, 32), _u8(4, 2)), "not implemented for 'Int'"),
    (lambda x: _C.mxfp4_dequant(x, _u8(4, 16), _u8(4, 2)), "expected 4 rows of 32"),
])
def test_quant_refusals(call, match):
    with pytest.raises(RuntimeError, match=match):
        call(torch.zeros(4, 64, dtype=BF))


@pytest.mark.parametrize("change,match", [
    (dict(weight=torch.ones(64)), "weight must have the input dtype"),
    (dict(weight=torch.ones(32, dtype=BF)), "weight has 32 elements"),
    (dict(residual=torch.zeros(4, 64, dtype=BF)), "go together"),
    (dict(after_res=torch.zeros(4, 64, dtype=BF)), "go together"),
    (dict(residual=torch.zeros(4, 64), after_res=torch.zeros(4, 64, dtype=BF)),
     "residual must have the input dtype"),
    (dict(residual=torch.zeros(4, 64, dtype=BF), after_res=torch.zeros(3, 64, dtype=BF)),
     "after_res has 192 elements"),
    (dict(input=torch.zeros(64, 4, dtype=BF).t()), "input must be contiguous"),
    (dict(scale=_u8(2, 4)), "expected 4 rows of 2"),
])
def test_norm_quant_refusals(change, match):
    args = dict(result=_u8(4, 32), input=torch.zeros(4, 64, dtype=BF),
                weight=torch.ones(64, dtype=BF), scale=_u8(4, 2), epsilon=1e-6)
    with pytest.raises(RuntimeError, match=match):
        _C.rms_norm_mxfp4_quant(**(args | change))


@pytest.mark.parametrize("change,match", [
    (dict(result=torch.zeros(4, 8, dtype=torch.int32)), "not implemented for 'Int'"),
    (dict(result=torch.zeros(4, 7, dtype=BF)), "expected 4 rows of 8"),
    (dict(result=torch.zeros(8, 4, dtype=BF).t()), "result must be contiguous"),
    (dict(b=_u8(8, 48), b_scale=_u8(8, 3)), "expected 8 rows of 32"),
    (dict(b=_u8(2, 4, 32)), r"b must be \[N, K / 2\]"),
    (dict(a=_u8(4, 8), a_scale=_u8(4, 1)), "multiple of the block of 32"),
    (dict(a_scale=_u8(4, 1)), "scale of a has shape"),
    (dict(bias=torch.zeros(8)), "bias must have the result dtype"),
    (dict(bias=torch.zeros(4, dtype=BF)), "bias has 4 elements"),
])
def test_product_refusals(change, match):
    args = dict(result=torch.zeros(4, 8, dtype=BF), a=_u8(4, 32), a_scale=_u8(4, 2),
                b=_u8(8, 32), b_scale=_u8(8, 2))
    with pytest.raises(RuntimeError, match=match):
        _C.mxfp4_scaled_mm(**(args | change))


def _cache(kind="int8", pages=3, page=16, heads=2, dim=64):
    if kind == "mxfp4":
        return _u8(pages, page, heads, dim // 2), _u8(pages, page, heads, dim // 32)
    dtype = torch.int8 if kind == "int8" else torch.float8_e4m3fn
    return (torch.zeros(pages, page, heads, dim).to(dtype), torch.zeros(pages, page, heads))


_KV = torch.zeros(4, 2, 64, dtype=BF)


@pytest.mark.parametrize("change,match", [
    (dict(key=_KV.int(), value=_KV.int()), "not implemented for 'Int'"),
    (dict(value=_KV.float()), "value must have key's dtype"),
    (dict(value=_KV[:3]), "the same tokens and heads"),
    (dict(key=torch.zeros(4, 128, dtype=BF)), "the same tokens and heads"),
    (dict(key=torch.zeros(4, 64, 2, dtype=BF).transpose(1, 2)), "must be contiguous"),
    (dict(slot_mapping=torch.zeros(4, dtype=torch.int32)), "slot_mapping must be"),
    (dict(slot_mapping=torch.zeros(5, dtype=torch.int64)), "at most one slot a token"),
    (dict(key_cache=_cache()[0].float()), "the caches must share a dtype"),
    (dict(key_cache=_cache()[0].float(), value_cache=_cache()[0].float()), "the cache must be int8"),
    (dict(key_cache=_cache(dim=32)[0]), "beside"),
    (dict(value_cache=_cache(page=8)[0]), "the caches' shapes differ"),
    (dict(key_scale=torch.zeros(3, 16)), "scale of key has shape"),
    (dict(key_scale=torch.zeros(3, 16, 2, dtype=BF)), "must be float32"),
    (dict(key_cache=_cache(page=1)[0].expand(3, 16, 2, 64)), "share memory"),
    (dict(key_scale=torch.zeros(3, 1, 2).expand(3, 16, 2)), "share memory"),
])
def test_cache_write_refusals(change, match):
    codes, scale = _cache()
    args = dict(key=_KV, value=_KV, key_cache=codes, value_cache=codes.clone(), key_scale=scale,
                value_scale=scale.clone(), slot_mapping=torch.zeros(4, dtype=torch.int64))
    with pytest.raises(RuntimeError, match=match):
        _C.kv_cache_write_quant(**(args | change))


def test_four_bit_cache_refusals():
    codes, scale = _cache("mxfp4", dim=96)
    kv = torch.zeros(4, 2, 96, dtype=BF)
    slots = torch.zeros(4, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="scale of key has shape"):
        _C.kv_cache_write_quant(kv, kv, codes, codes, torch.zeros(3, 16, 2), scale, slots)
    with pytest.raises(RuntimeError, match="must be uint8 or float8_e8m0fnu"):
        _C.kv_cache_write_quant(kv, kv, codes, codes, scale.float(), scale, slots)
    with pytest.raises(RuntimeError, match="multiple of the block of 32"):
        _C.kv_cache_write_quant(kv[..., :80].contiguous(), kv, codes[..., :40], codes, scale,
                                scale, slots)
    with pytest.raises(RuntimeError, match="CUDA"):  # nothing else is wrong with it
        _C.kv_cache_write_quant(kv, kv, codes, codes, scale, scale, slots)


@pytest.mark.parametrize("change,match", [
    (dict(block_table=torch.zeros(1, 3, dtype=torch.int64)), "block_table must be"),
    (dict(block_table=torch.zeros(3, dtype=torch.int32)), r"\[sequences, pages\]"),
    (dict(block_table=torch.zeros(3, 1, dtype=torch.int32).t().expand(1, 3)[:, ::2]),
     "contiguous rows"),
    (dict(cu_seqlens=torch.zeros(3, dtype=torch.int32)), "with 2 elements"),
    (dict(cu_seqlens=torch.zeros(2, dtype=torch.int64)), "cu_seqlens must be"),
    (dict(seq_starts=torch.zeros(2, dtype=torch.int32)), "with 1 elements"),
    (dict(key=torch.zeros(1, 2, 64, dtype=BF).expand(4, 2, 64)), "share memory"),
])
def test_cache_read_refusals(change, match):
    codes, scale = _cache("fp8")
    args = dict(key=_KV, value=_KV.clone(), key_cache=codes, value_cache=codes, key_scale=scale,
                value_scale=scale, block_table=torch.zeros(1, 3, dtype=torch.int32),
                cu_seqlens=torch.zeros(2, dtype=torch.int32))
    with pytest.raises(RuntimeError, match=match):
        _C.kv_cache_read_dequant(**(args | change))


def _side(**change):
    side = dict(plain=16, token_stride=128, head_stride=64, codes=16, code_page_stride=2048,
                code_token_stride=128, code_head_stride=64, scales=16, scale_page_stride=32,
                scale_token_stride=2, scale_head_stride=1, head_size=64)
    return _lib.KvSide(**(side | change))


def test_c_abi_refuses_bad_arguments_without_a_device():
    lib, p = _lib.lib, ctypes.c_void_p(16)  # never dereferenced

    def refused(rc, text, code=-1):
        assert rc == code and text in lib.mcop_last_error().decode(), (rc, lib.mcop_last_error())

    assert lib.mcop_mxfp4_quant(None, None, None, 0, 64, 64, 0, None) == 0
    refused(lib.mcop_mxfp4_quant(p, p, p, 4, 0, 64, 0, None), "bad shape")
    refused(lib.mcop_mxfp4_quant(p, p, p, 4, 48, 48, 0, None), "multiple of the block")
    refused(lib.mcop_mxfp4_quant(p, None, p, 4, 64, 64, 0, None), "null pointer")
    refused(lib.mcop_mxfp4_quant(p, p, p, 4, 64, -1, 0, None), "input_row_stride")
    refused(lib.mcop_mxfp4_quant(p, p, p, 4, 64, 64, 3, None), "input dtype")
    refused(lib.mcop_mxfp4_quant(ctypes.c_void_p(18), p, p, 4, 64, 64, 0, None), "aligned")
    refused(lib.mcop_mxfp4_quant(p, p, p, 1 << 60, 64, 64, 0, None), "bad shape")
    refused(lib.mcop_mxfp4_dequant(p, 4, p, p, 4, 64, None), "out dtype")
    refused(lib.mcop_rms_norm_mxfp4_quant(p, p, p, p, p, None, 4, 64, 0, 1e-6, None), "go together")
    refused(lib.mcop_rms_norm_mxfp4_quant(p, p, p, p, None, None, 4, 64, 5, 1e-6, None),
            "input dtype")
    refused(lib.mcop_rms_norm_mxfp4_quant(p, p, p, p, None, None, 4, 100, 0, 1e-6, None),
            "multiple of the block")
    refused(lib.mcop_mxfp4_scaled_mm(p, 0, p, p, p, p, None, 4, 8, 40, None),
            "multiple of the block")
    refused(lib.mcop_mxfp4_scaled_mm(p, 3, p, p, p, p, None, 4, 8, 64, None), "out dtype")
    refused(lib.mcop_mxfp4_scaled_mm(p, 0, ctypes.c_void_p(24), p, p, p, None, 4, 8, 64, None),
            "aligned to 16")
    refused(lib.mcop_mxfp4_scaled_mm(p, 0, p, p, p, p, None, 1 << 40, 8, 64, None), "one launch", -2)
    refused(lib.mcop_mxfp4_scaled_mm(p, 0, p, p, p, p, None, 4, 1 << 28, 64, None), "one launch", -2)
    assert lib.mcop_mxfp4_scaled_mm(None, 0, None, None, None, None, None, 0, 8, 64, None) == 0

    def write(k, v, fmt=3, pages=2, page=16, heads=2, tokens=4, dtype=0, slots=p):
        return lib.mcop_kv_cache_write_quant(ctypes.byref(k), ctypes.byref(v), fmt, pages, page,
                                             heads, slots, tokens, dtype, None)

    good = _side()
    assert write(good, good, tokens=0) == 0 and write(good, good, pages=0) == 0
    refused(write(good, good, fmt=0), "cache dtype")
    refused(write(good, good, dtype=3), "dtype 3 is not")
    refused(write(good, good, heads=0), "bad shape")
    refused(write(good, good, pages=1 << 30, page=2), "2^31 - 1 slots")
    refused(write(good, good, tokens=1 << 31), "2^31 vectors", -2)
    refused(write(good, good, slots=None), "null pointer")
    # 2^32 threads or more: 2^30 vectors of 8 lanes, and four times 2^26 vectors of 64 lanes by fours
    refused(write(good, good, tokens=1 << 29), "one launch", -2)
    refused(write(_side(head_size=512), good, tokens=1 << 28), "one launch", -2)
    wide = _side(head_size=512)
    refused(write(wide, wide, tokens=1 << 27), "one launch", -2)
    refused(write(_side(head_size=0), good), "key head_size 0")
    refused(write(good, _side(head_size=1025)), "value head_size 1025")
    refused(write(_side(head_size=48), good, fmt=5), "multiple of the block")
    refused(write(_side(code_page_stride=-1), good), "bad key stride")
    refused(write(_side(codes=None), good), "null pointer")

    def read(table=p, columns=2, stride=2, cu=p, sequences=1, tokens=4):
        return lib.mcop_kv_cache_read_dequant(ctypes.byref(good), ctypes.byref(good), 3, 2, 16, 2,
                                              table, stride, columns, cu, None, sequences, tokens, 0,
                                              None)

    assert read(tokens=0) == 0 and read(sequences=0) == 0
    refused(read(cu=None), "null pointer")
    refused(read(table=None), "null pointer")
    refused(read(sequences=-1), "bad block table")
    refused(read(stride=-1), "bad block table")


def test_the_plain_format_is_its_own_inverse():
    """Codes of values that are codes give the same codes, with the scale of the largest."""
    for code in range(1, 16):
        if code == 8:
            continue  # -0 alone: a block of zeros
        block = torch.zeros(BLOCK := 32, dtype=torch.uint8)
        block[5] = code
        v = mx_plain.values(block[None], torch.tensor([[130]], dtype=torch.uint8))
        got, byte = mx_plain.quant(v.float())
        assert torch.equal(mx_plain.values(got, byte), v) and BLOCK == 32
