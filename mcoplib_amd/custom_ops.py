"""``mcoplib.custom_ops`` wrappers of the fused norm/quant path (reference
mcoplib/custom_ops.py:7-45): allocate the outputs the way the reference does and call the
``op`` entry point, both in the _torch_ops extension.  The 4-bit operators and the quantized
key/value cache, which the reference does not have, are here in the same manner."""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import op as ops  # noqa: F401  (loads the library, then the extension)
from . import _torch_ops


def fused_add_rms_norm_dynamic_per_token_quant_padding_output(
        input: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, pad_size: int,
        epsilon: float):
    """Allocates the padded output as bf16 [..., pad_size] (2*pad_size bytes per row, viewed as
    int8 for the kernel), output_rms like input, the unpacked int8 codes and scales [T, 1], and
    returns (output, residual, output_rms, output_quant_int8, scales); ``residual`` is updated
    in place (reference mcoplib/custom_ops.py:7-27)."""
    assert input.is_contiguous()
    assert weight.is_contiguous()
    return _torch_ops.padded_new(input, residual, weight, pad_size, epsilon)


def rms_norm_dynamic_per_token_quant(input: torch.Tensor, weight: torch.Tensor, epsilon: float,
                                     quant_dtype: torch.dtype,
                                     scale_ub: Optional[torch.Tensor] = None,
                                     residual: Optional[torch.Tensor] = None
                                     ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Returns (codes like input in quant_dtype, scales [T, 1] fp32); updates ``residual`` in
    place when given.  ``quant_dtype`` must be int8, as for the reference custom op."""
    return _torch_ops.custom_new(input, weight, epsilon, quant_dtype, scale_ub, residual)


def mxfp4_quant(input: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Returns (codes [..., H / 2], scales [..., H / 32]), both uint8, of rows of H values (a multiple
    of 32; bf16, fp16 or fp32; rows may be strided).  Value 2i of a row is the low half of byte i, a
    code e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign); a scale byte e is 2^(e - 127).  A block of 32
    that holds a NaN or an infinity reads back as NaN (e = 255)."""
    return _torch_ops.mxfp4_quant_new(input)


def mxfp4_dequant(codes: torch.Tensor, scale: torch.Tensor, out_dtype: torch.dtype) -> torch.Tensor:
    """The values of mxfp4_quant's codes and scales, rounded once to out_dtype."""
    return _torch_ops.mxfp4_dequant_new(codes, scale, out_dtype)


def rms_norm_mxfp4_quant(input: torch.Tensor, weight: torch.Tensor, epsilon: float,
                         residual: Optional[torch.Tensor] = None
                         ) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """Returns (codes, scales, after_res): mxfp4_quant of the normalized rows of input (+ residual),
    and input + residual in a new tensor (None without a residual, which is not changed).  To add in
    place, pass the residual as after_res to torch.ops._C.rms_norm_mxfp4_quant."""
    return _torch_ops.rms_norm_mxfp4_quant_new(input, weight, epsilon, residual)


def mxfp4_scaled_mm(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor,
                    out_dtype: torch.dtype, bias: Optional[torch.Tensor] = None) -> torch.Tensor:
    """a [..., K / 2] times the transpose of b [N, K / 2], both as mxfp4_quant gives them, plus bias
    [N] (of out_dtype): summed in fp32, rounded once to out_dtype (bf16, fp16 or fp32)."""
    return _torch_ops.mxfp4_scaled_mm_new(a, a_scale, b, b_scale, out_dtype, bias)


def kv_cache_write_quant(key: torch.Tensor, value: torch.Tensor, key_cache: torch.Tensor,
                         value_cache: torch.Tensor, key_scale: torch.Tensor,
                         value_scale: torch.Tensor, slot_mapping: torch.Tensor) -> None:
    """Quantizes key and value [tokens, heads, head_size] (any strides but the last) into the slots
    (page * page_size + offset; int64) of a paged cache [pages, page_size, heads, head_size]: int8 or
    float8_e4m3fn with fp32 scales [pages, page_size, heads], one a token and head, or 4-bit codes,
    uint8 [..., head_size / 2] with uint8 scales [..., head_size / 32].  slot_mapping may cover fewer
    tokens than key has; negative slots (padding) and slots past the cache are not written.  Slots that
    are written must differ from each other, and the caches and scales must not overlap."""
    _torch_ops.c_kv_cache_write_quant(key, value, key_cache, value_cache, key_scale, value_scale,
                                      slot_mapping)


def kv_cache_read_dequant(key_cache: torch.Tensor, value_cache: torch.Tensor,
                          key_scale: torch.Tensor, value_scale: torch.Tensor,
                          block_table: torch.Tensor, cu_seqlens: torch.Tensor, num_tokens: int,
                          out_dtype: torch.dtype, seq_starts: Optional[torch.Tensor] = None
                          ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Returns (key, value) [num_tokens, heads, head_size] in out_dtype: rows cu_seqlens[s] to
    cu_seqlens[s + 1] are the positions from seq_starts[s] (or 0) on of sequence s, whose pages
    block_table[s] lists (all int32).  num_tokens is the host's count of the rows, cu_seqlens[-1];
    rows past that are not written.  A position without a page of the cache reads as NaN."""
    return _torch_ops.kv_cache_read_new(key_cache, value_cache, key_scale, value_scale, block_table,
                                        cu_seqlens, num_tokens, out_dtype, seq_starts)
