"""Without a GPU: the schemas, Meta kernels and refusals of the cache's attention and of its page operators,
on their surfaces and in the C ABI, and the tests' own plain pool."""

import ctypes

import pytest
import torch

import kv_plain
import mcoplib._C  # noqa: F401
from mcoplib import custom_ops
from mcoplib_amd import _C, _lib

BF = torch.bfloat16
I32 = torch.int32


def _ints(*values):
    return torch.tensor(values, dtype=I32)


def test_schemas_name_their_outputs():
    writes = {"kv_cache_attention": ["result", "lse"], "kv_cache_copy_pages": ["caches"],
              "kv_cache_fork": ["block_table", "seq_lens", "ref_counts", "src", "dst"],
              "kv_cache_extend": ["block_table", "seq_lens", "ref_counts", "slots", "starts"],
              "kv_cache_free": ["block_table", "seq_lens", "ref_counts"],
              "kv_cache_compact": ["block_table", "ref_counts", "src", "dst", "used"]}
    for name, outs in writes.items():
        schema = getattr(torch.ops._C, name).default._schema
        assert [a.name for a in schema.arguments
                if a.alias_info is not None and a.alias_info.is_write] == outs, name
        assert not schema.returns


def test_meta_kernels_accept_meta_tensors():
    m = torch.device("meta")
    e = lambda *s, dtype=I32: torch.empty(*s, dtype=dtype, device=m)  # noqa: E731
    q, cache, scale = e(4, 8, 64, dtype=BF), e(3, 16, 2, 64, dtype=torch.int8), e(3, 16, 2, dtype=torch.float)
    ops = torch.ops._C
    ops.kv_cache_attention(q, q, cache, cache, scale, scale, e(4, 2), e(4), 0.125, 0, None)
    ops.kv_cache_copy_pages([cache, scale], e(2), e(2))
    ops.kv_cache_fork(e(4, 2), e(4), e(3), e(1), e(1), e(1), e(1), 16)
    ops.kv_cache_extend(e(4, 2), e(4), e(3), e(1), e(2), e(5, dtype=torch.int64), e(1), 16)
    ops.kv_cache_free(e(4, 2), e(4), e(3), e(1), 16)
    ops.kv_cache_compact(e(4, 2), e(3), e(1), e(1), e(1))


def _attention_args(kind="int8", **change):
    codes = {"int8": torch.int8, "fp8": torch.float8_e4m3fn, "mxfp4": torch.uint8}[kind]
    width, tail = (32, (2,)) if kind == "mxfp4" else (64, ())
    scale = torch.uint8 if kind == "mxfp4" else torch.float32
    args = dict(result=torch.zeros(4, 8, 64, dtype=BF), query=torch.zeros(4, 8, 64, dtype=BF),
                key_cache=torch.zeros(3, 16, 2, width).to(codes),
                value_cache=torch.zeros(3, 16, 2, width).to(codes),
                key_scale=torch.zeros(3, 16, 2, *tail, dtype=scale),
                value_scale=torch.zeros(3, 16, 2, *tail, dtype=scale),
                block_table=torch.zeros(4, 3, dtype=I32), seq_lens=torch.zeros(4, dtype=I32), scale=0.125)
    return args | change


@pytest.mark.parametrize("change,match", [
    (dict(query=torch.zeros(4, 8, 64, dtype=I32)), "not implemented for 'Int'"),
    (dict(result=torch.zeros(4, 8, 64)), "result must have query's dtype"),
    (dict(result=torch.zeros(3, 8, 64, dtype=BF)), "same sequences and heads"),
    (dict(query=torch.zeros(4, 512, dtype=BF)), "same sequences and heads"),
    (dict(query=torch.zeros(4, 7, 64, dtype=BF), result=torch.zeros(4, 7, 64, dtype=BF)),
     "7 query heads are not a multiple of 2"),
    (dict(query=torch.zeros(4, 0, 64, dtype=BF), result=torch.zeros(4, 0, 64, dtype=BF)),
     "0 query heads are not a multiple of 2"),
    (dict(query=torch.zeros(4, 8, 32, dtype=BF)), "beside"),
    (dict(result=torch.zeros(4, 8, 32, dtype=BF)), "beside"),
    (dict(query=torch.zeros(4, 64, 8, dtype=BF).transpose(1, 2)), "must be contiguous"),
    (dict(value_cache=torch.zeros(3, 16, 2, 64)), "the caches must share a dtype"),
    (dict(key_cache=torch.zeros(3, 16, 2, 64), value_cache=torch.zeros(3, 16, 2, 64)),
     "the cache must be int8"),
    (dict(value_cache=torch.zeros(3, 8, 2, 64, dtype=torch.int8)), "the caches' shapes differ"),
    (dict(key_scale=torch.zeros(3, 16)), "scale of key has shape"),
    (dict(value_scale=torch.zeros(3, 16, 2, dtype=BF)), "must be float32"),
    (dict(block_table=torch.zeros(3, 3, dtype=I32)), "block_table has 3 rows for 4"),
    (dict(block_table=torch.zeros(4, 3, dtype=torch.int64)), "block_table must be"),
    (dict(block_table=torch.zeros(3, 4, dtype=I32).t()), "contiguous rows"),
    (dict(seq_lens=torch.zeros(3, dtype=I32)), "seq_lens must be contiguous with 4 elements"),
    (dict(seq_lens=torch.zeros(4, dtype=torch.int64)), "seq_lens must be"),
    (dict(seq_lens=torch.zeros(8, dtype=I32)[::2]), "seq_lens must be contiguous"),
    (dict(window=-1), "window must not be negative"),
    (dict(lse=torch.zeros(4, 8, dtype=BF)), "lse must be contiguous float32"),
    (dict(lse=torch.zeros(8, 4).t()), "lse must be contiguous float32"),
    (dict(result=torch.zeros(4, 1, 64, dtype=BF).expand(4, 8, 64)), "share memory"),
    (dict(), "CUDA"),
])
def test_attention_refusals(change, match):
    with pytest.raises(RuntimeError, match=match):
        _C.kv_cache_attention(**_attention_args(**change))


def test_attention_refusals_of_the_allocating_form():
    args = _attention_args("mxfp4")
    del args["result"]
    with pytest.raises(RuntimeError, match="CUDA"):
        custom_ops.kv_cache_attention(**args)
    with pytest.raises(RuntimeError, match="query must be"):
        custom_ops.kv_cache_attention(**(args | dict(query=torch.zeros(4, 64, dtype=BF))))
    with pytest.raises(RuntimeError, match="multiple of the block of 32"):
        custom_ops.kv_cache_attention(**(args | dict(query=torch.zeros(4, 8, 48, dtype=BF))))


@pytest.mark.parametrize("caches,src,dst,match", [
    ([torch.zeros(4, 3)], _ints(0).long(), _ints(1), "src must be"),
    ([torch.zeros(4, 3)], _ints(0, 1), _ints(1), "dst must be contiguous with 2 elements"),
    ([torch.zeros(4, 3)], _ints(0, 1, 2, 3)[::2], _ints(1, 2), "src must be contiguous"),
    ([torch.zeros(4, 3)], _ints(0), _ints(1), "CUDA"),
    ([torch.zeros(())], _ints(0), _ints(1), "the same pages"),
    ([torch.zeros(4, 3), torch.zeros(5, 3)], _ints(0), _ints(1), "CUDA|the same pages"),
])
def test_copy_refusals(caches, src, dst, match):
    with pytest.raises(RuntimeError, match=match):
        _C.kv_cache_copy_pages(caches, src, dst)


def _pool(**change):
    args = dict(block_table=torch.zeros(4, 3, dtype=I32), seq_lens=_ints(0, 0, 0, 0),
                ref_counts=torch.zeros(9, dtype=I32))
    return args | change


@pytest.mark.parametrize("change,match", [
    (dict(block_table=torch.zeros(4, 3)), "block_table must be"),
    (dict(block_table=torch.zeros(4, dtype=I32)), r"\[sequences, pages\]"),
    (dict(block_table=torch.zeros(4, 6, dtype=I32)[:, ::2]), "contiguous rows"),
    (dict(block_table=torch.zeros(1, 3, dtype=I32).expand(4, 3)), "share memory"),
    (dict(seq_lens=_ints(0, 0, 0)), "seq_lens must be contiguous with 4"),
    (dict(ref_counts=torch.zeros(9)), "ref_counts must be"),
    (dict(ref_counts=torch.zeros(3, 3, dtype=I32)), "ref_counts must be contiguous"),
    (dict(page_size=0), "page_size must be positive"),
    (dict(), "CUDA"),
])
def test_pool_refusals(change, match):
    size = dict(page_size=16)
    with pytest.raises(RuntimeError, match=match):
        custom_ops.kv_cache_free(**(_pool() | size | dict(sequences=_ints(1)) | change))
    with pytest.raises(RuntimeError, match=match):
        custom_ops.kv_cache_fork(**(_pool() | size | dict(parents=_ints(1), children=_ints(2)) | change))
    with pytest.raises(RuntimeError, match=match):
        custom_ops.kv_cache_extend(**(_pool() | size | dict(sequences=_ints(1), cu_tokens=_ints(0, 2),
                                                            num_tokens=2) | change))
    if "seq_lens" not in change and "page_size" not in change:
        pool = _pool() | change
        with pytest.raises(RuntimeError, match=match):
            custom_ops.kv_cache_compact(pool["block_table"], pool["ref_counts"])


def test_request_refusals():
    with pytest.raises(RuntimeError, match="children must be contiguous with 2"):
        custom_ops.kv_cache_fork(**_pool(), parents=_ints(1, 2), children=_ints(3), page_size=16)
    with pytest.raises(RuntimeError, match="cu_tokens must be contiguous with 3"):
        custom_ops.kv_cache_extend(**_pool(), sequences=_ints(1, 2), cu_tokens=_ints(0, 3), num_tokens=3,
                                   page_size=16)
    with pytest.raises(RuntimeError, match="num_tokens must not be negative"):
        custom_ops.kv_cache_extend(**_pool(), sequences=_ints(1), cu_tokens=_ints(0, 3), num_tokens=-1,
                                   page_size=16)
    with pytest.raises(RuntimeError, match="slots must be"):
        _C.kv_cache_extend(**_pool(), sequences=_ints(1), cu_tokens=_ints(0, 3), slots=_ints(0, 0, 0),
                           starts=_ints(0), page_size=16)
    with pytest.raises(RuntimeError, match="src must be contiguous with 4"):
        _C.kv_cache_compact(torch.zeros(4, 3, dtype=I32), torch.zeros(9, dtype=I32), _ints(0, 0, 0),
                            _ints(0, 0, 0, 0), _ints(0))


def _side(**change):
    side = dict(plain=16, token_stride=512, head_stride=64, codes=16, code_page_stride=2048,
                code_token_stride=128, code_head_stride=64, scales=16, scale_page_stride=32,
                scale_token_stride=2, scale_head_stride=1, head_size=64)
    return _lib.KvSide(**(side | change))


def test_the_attention_entry_refuses_bad_arguments_without_a_device():
    lib, p = _lib.lib, ctypes.c_void_p(16)  # never dereferenced

    def refused(rc, text, code=-1):
        assert rc == code and text in lib.mcop_last_error().decode(), (rc, lib.mcop_last_error())

    room = lib.mcop_kv_cache_attention_workspace(2, 8, 64)
    assert room > 0
    assert lib.mcop_kv_cache_attention_workspace(3, 8, 64) == -1
    assert lib.mcop_kv_cache_attention_workspace(2, 8, 1025) == -1
    assert lib.mcop_kv_cache_attention_workspace(1, 65536, 64) == -1

    def call(k=None, v=None, fmt=3, pages=2, page=16, heads=2, queries=8, table=p, stride=3, columns=3,
             lens=p, sequences=4, window=0, dtype=0, ws=p, room=room):
        k, v = k or _side(), v or _side()
        return lib.mcop_kv_cache_attention(ctypes.byref(k), ctypes.byref(v), fmt, pages, page, heads, queries,
                                           table, stride, columns, lens, sequences, 0.1, window, dtype, None,
                                           ws, room, None)

    assert call(sequences=0) == 0
    refused(call(fmt=0), "cache dtype")
    refused(call(dtype=3), "dtype 3 is not")
    refused(call(heads=0), "query heads")
    refused(call(queries=7), "query heads")
    refused(call(heads=1, queries=65536), "query heads")
    refused(call(page=0), "bad shape")
    refused(call(pages=1 << 30, page=2), "2^31 - 1 slots")
    refused(call(sequences=-1), "bad block table")
    refused(call(sequences=(1 << 24) + 1), "bad block table")
    refused(call(stride=-1), "bad block table")
    refused(call(sequences=1 << 20, columns=1 << 20), "2^31 tiles", -2)
    refused(call(window=-1), "negative window")
    refused(call(k=_side(head_size=0)), "key head_size 0")
    refused(call(v=_side(head_size=1025)), "value head_size 1025")
    refused(call(k=_side(head_size=48), fmt=5), "multiple of the block")
    refused(call(v=_side(codes=None)), "null pointer")
    refused(call(lens=None), "null pointer")
    refused(call(table=None), "null pointer")
    refused(call(ws=None), "workspace must be")
    refused(call(ws=ctypes.c_void_p(24)), "workspace must be")
    refused(call(room=room - 1), "workspace must be")
    assert lib.mcop_kv_cache_attention(None, None, 3, 2, 16, 2, 8, p, 3, 3, p, 4, 0.1, 0, 0, None, p, room,
                                       None) == -1


def test_the_page_entries_refuse_bad_arguments_without_a_device():
    lib, p = _lib.lib, ctypes.c_void_p(16)

    def refused(rc, text, code=-1):
        assert rc == code and text in lib.mcop_last_error().decode(), (rc, lib.mcop_last_error())

    def pool(**change):
        d = dict(block_table=16, table_row_stride=3, num_rows=4, table_columns=3, seq_lens=16, ref_counts=16,
                 num_pages=9, page_size=16)
        return ctypes.byref(_lib.KvPool(**(d | change)))

    room = lib.mcop_kv_cache_pages_workspace(2, 9)
    assert room == 4 * (4 + 2 + 9)
    assert lib.mcop_kv_cache_pages_workspace(-1, 9) == -1
    assert lib.mcop_kv_cache_pages_workspace(1, 1 << 31) == -1

    def fork(q, n=2, src=p, ws=p, room=room):
        return lib.mcop_kv_cache_fork(q, p, p, n, src, p, ws, room, None)

    assert fork(pool(), n=0) == 0
    refused(fork(None), "null pointer")
    for change in (dict(num_rows=-1), dict(table_columns=-1), dict(table_row_stride=-1), dict(num_pages=-1),
                   dict(num_pages=1 << 31), dict(page_size=0), dict(num_rows=1 << 31)):
        refused(fork(pool(**change)), "bad pool")
    for name in ("block_table", "seq_lens", "ref_counts"):
        refused(fork(pool(**{name: None})), "null pointer")
    refused(fork(pool(), src=None), "null pointer")
    refused(fork(pool(), n=-1), "bad number of requests")
    refused(fork(pool(), n=1 << 24), "bad number of requests")
    refused(fork(pool(), room=room - 1), "workspace must be")
    refused(fork(pool(), ws=ctypes.c_void_p(20)), "workspace must be")

    def extend(q, n=2, tokens=5, slots=p, starts=p, room=room):
        return lib.mcop_kv_cache_extend(q, p, p, n, slots, tokens, starts, p, room, None)

    assert extend(pool(), n=0, tokens=0) == 0
    refused(extend(pool(), tokens=-1), "num_tokens")
    refused(extend(pool(), slots=None), "null pointer")
    refused(extend(pool(), starts=None), "null pointer")
    refused(extend(pool(), room=8), "workspace must be")
    assert lib.mcop_kv_cache_free(pool(), p, 0, None) == 0
    refused(lib.mcop_kv_cache_free(pool(), None, 1, None), "null pointer")
    refused(lib.mcop_kv_cache_free(pool(seq_lens=None), p, 1, None), "null pointer")

    def compact(q, src=p, used=p, room=4 * (4 + 9)):
        return lib.mcop_kv_cache_compact(q, src, p, used, p, room, None)

    refused(compact(pool(), src=None), "null pointer")
    refused(compact(pool(), used=None), "null pointer")
    refused(compact(pool(), room=16), "workspace must be")
    refused(compact(pool(num_rows=1 << 17, table_columns=1 << 15, table_row_stride=1 << 15)), "one launch", -2)

    def copy(tensors, pages=4, pairs=2, src=p):
        array = (_lib.KvPages * len(tensors))(*(_lib.KvPages(*t) for t in tensors))
        return lib.mcop_kv_cache_copy_pages(array, len(tensors), pages, src, p, pairs, None)

    assert copy([(16, 64, 64)], pairs=0) == 0 and copy([(16, 64, 64)], pages=0) == 0
    refused(copy([(16, 64, 64)], pairs=-1), "bad shape")
    refused(copy([(16, 64, 64)], src=None), "null pointer")
    refused(copy([(16, 64, 64), (None, 64, 64)]), "tensor 1")
    refused(copy([(16, 0, 64)]), "tensor 0")
    refused(copy([(16, 64, 63)]), "tensor 0")
    refused(copy([(16, 64, 1 << 62)]), "tensor 0")
    refused(copy([(16, 1 << 40, 1 << 40)]), "one launch", -2)


def test_the_plain_pool_gives_back_what_it_takes():
    pool = kv_plain.PagePool(torch.full((5, 4), -1), torch.zeros(5, dtype=I32), torch.zeros(9, dtype=I32), 4)
    slots, starts = pool.extend([0, 1], [0, 6, 7], 8)
    assert slots == [0, 1, 2, 3, 4, 5, 8, -1] and starts == [0, 0]
    assert pool.fork([0, 0], [2, 3]) == ([1, 1], [3, 4])
    assert pool.counts == [3, 1, 1, 1, 1, 0, 0, 0, 0]
    assert pool.extend([2], [0, 20], 20)[1] == [-1]  # past its row
    pool.free([0, 1, 1])
    assert pool.counts == [2, 0, 0, 1, 1, 0, 0, 0, 0]
    assert pool.compact() == ([4, 3, -1, -1], [1, 2, -1, -1], [3])
    assert pool.counts == [2, 1, 1, 0, 0, 0, 0, 0, 0]
    pool.free([2, 3])
    assert sum(pool.counts) == 0 and all(p == -1 for row in pool.table for p in row)
