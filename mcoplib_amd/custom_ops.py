"""``mcoplib.custom_ops`` wrappers of the fused norm/quant path (reference
mcoplib/custom_ops.py:7-45): allocate the outputs the way the reference does and call the
``op`` entry point, both in the _torch_ops extension.  The 4-bit operators, the quantized
key/value cache, attention over it and its pages, which the reference does not have, are here in the
same manner."""

from __future__ import annotations

from typing import Optional, Sequence, Tuple, Union

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


def kv_cache_attention(query: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                       key_scale: torch.Tensor, value_scale: torch.Tensor,
                       block_table: torch.Tensor, seq_lens: torch.Tensor,
                       scale: Optional[float] = None, window: int = 0, return_lse: bool = False
                       ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Attention of one new token a sequence over the cache that kv_cache_write_quant fills: query
    [sequences, query heads, head_size] (any strides but the last; query heads a multiple of the cache's
    heads, query head h reads head h // (query heads // heads)) over positions max(0, n - window)
    (window 0: from 0) to n - 1 of each sequence, n = seq_lens[s] (int32, the new token included), whose
    pages block_table[s] lists.  scale is head_size ** -0.5 where it is None.  Returns the outputs
    [sequences, query heads, value head_size] in query's dtype, with return_lse also the log of each
    row's sum of e^(scale q k) in fp32 [sequences, query heads], for a join with other positions.  A
    sequence of no positions gives 0 and -inf; one with a position without a page of the cache gives
    NaN.  Lengths are read on the device: a captured graph replays with new ones."""
    out, lse = _torch_ops.kv_cache_attention_new(query, key_cache, value_cache, key_scale, value_scale,
                                                 block_table, seq_lens, scale, window, return_lse)
    return (out, lse) if return_lse else out


def kv_cache_copy_pages(caches: Sequence[torch.Tensor], src: torch.Tensor, dst: torch.Tensor) -> None:
    """Copies page src[i] to page dst[i] (int32) in every tensor [pages, ...] of caches: the codes and
    scales of every layer, in one launch for 64 of them.  A page's elements must lie together.  Pairs with
    a negative index or one past the pages are left out; pages that are written must differ from each
    other and from those that are read."""
    _torch_ops.c_kv_cache_copy_pages(caches, src, dst)


def kv_cache_fork(block_table: torch.Tensor, seq_lens: torch.Tensor, ref_counts: torch.Tensor,
                  parents: torch.Tensor, children: torch.Tensor, page_size: int
                  ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Forks sequences (rows of block_table [sequences, pages], with their lengths seq_lens and the pages'
    ref_counts [pages], 0 for a free page; all int32, all updated in place): children[i] becomes a copy of
    parents[i], which it shares the full pages of.  A last page that is filled in part is replaced by a
    free one, the lowest free page for the first fork that needs one and so on.  Returns (src, dst): that
    page of the parent and of the child, for kv_cache_copy_pages, -1 where there is none.  A page that the
    parent has not, the child has not either.  A fork that no page is left for leaves its child empty.
    Children must be free rows, different from each other and from all parents; a parent may have many."""
    return _torch_ops.kv_cache_fork_new(block_table, seq_lens, ref_counts, parents, children, page_size)


def kv_cache_extend(block_table: torch.Tensor, seq_lens: torch.Tensor, ref_counts: torch.Tensor,
                    sequences: torch.Tensor, cu_tokens: torch.Tensor, num_tokens: int,
                    page_size: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """Makes room for new tokens: sequences[i] grows by cu_tokens[i + 1] - cu_tokens[i] (int32, from 0),
    and takes the lowest free pages, in order of i.  num_tokens is the host's count of the new tokens,
    cu_tokens[-1].  Returns (slots, starts): slots [num_tokens] (int64) is the new tokens' slot_mapping for
    kv_cache_write_quant, starts [sequences] (int32) the first new position of each.  Where the free pages
    end, that sequence and those behind it that need a page stay as they are, as does one that would not
    fit its row or 32 bits: their starts and slots are -1, which kv_cache_write_quant does not write.  The
    pool's tensors are as in kv_cache_fork; sequences must differ from each other, and a sequence's part-filled
    last page must be its own (a fork's is)."""
    return _torch_ops.kv_cache_extend_new(block_table, seq_lens, ref_counts, sequences, cu_tokens,
                                          num_tokens, page_size)


def kv_cache_free(block_table: torch.Tensor, seq_lens: torch.Tensor, ref_counts: torch.Tensor,
                  sequences: torch.Tensor, page_size: int) -> None:
    """Gives back the pages of sequences (int32): each page is counted once less, the rows become -1 and
    the lengths 0.  A sequence that is named twice is given back once.  The pool's tensors are as in
    kv_cache_fork."""
    _torch_ops.c_kv_cache_free(block_table, seq_lens, ref_counts, sequences, page_size)


def kv_cache_compact(block_table: torch.Tensor, ref_counts: torch.Tensor
                     ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Moves the pages in use together, so that they are the first ones: those past their number go to the
    free ones below it, the highest to the lowest.  block_table and ref_counts are updated in place.
    Returns (src, dst, used): the moves [pages / 2], -1 behind the last, for kv_cache_copy_pages (which
    must follow, before the cache is used again), and the number of pages in use [1] (int32)."""
    return _torch_ops.kv_cache_compact_new(block_table, ref_counts)
