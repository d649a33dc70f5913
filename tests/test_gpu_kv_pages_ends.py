"""The page operators of the cache on the GPU where the pool's numbers end: forks of sequences whose last page is
missing, lengths next to 2^31."""

import pytest
import torch

import kv_plain
import mcoplib_amd._C  # noqa: F401
from gpu_util import DEV, gen, say
from mcoplib import custom_ops

pytestmark = pytest.mark.gpu


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _pool(rows, lens, pages, columns):
    """(block_table, seq_lens, ref_counts) on the device of sequences that share no page."""
    table = torch.full((len(rows), columns), -1, dtype=torch.int32)
    counts = torch.zeros(pages, dtype=torch.int32)
    for i, row in enumerate(rows):
        table[i, :len(row)] = torch.tensor(row, dtype=torch.int32)
        counts[[p for p in row if 0 <= p < pages]] = 1
    return table.to(DEV), _i32(lens), counts.to(DEV)


@pytest.mark.parametrize("columns", [4, 5000])  # in one launch, in two
@pytest.mark.parametrize("bad", [-1, 20, -(1 << 31), (1 << 31) - 1])
def test_forks_of_a_missing_last_page(bad, columns):
    """A part-filled page that the parent has not takes no free page, and its child has none."""
    say(f"forks of a last page {bad}, rows of {columns}")
    pool = _pool([[3, 7, bad], [5, 2], [], [], [], []], [21, 10, 0, 0, 0, 0], 20, columns)
    src, dst = custom_ops.kv_cache_fork(*pool, _i32([1, 0, 0, 1]), _i32([2, 3, 5, 4]), 8)
    assert src.tolist() == [2, -1, -1, 2] and dst.tolist() == [0, -1, -1, 1]
    table, lens, counts = (t.tolist() for t in pool)
    assert [row[:4] for row in table] == [[3, 7, bad, -1], [5, 2, -1, -1], [5, 0, -1, -1], [3, 7, -1, -1],
                                          [5, 1, -1, -1], [3, 7, -1, -1]]
    assert all(page == -1 for row in table for page in row[4:])
    assert lens == [21, 10, 10, 21, 10, 21]
    want = [0] * 20
    want[3] = want[7] = want[5] = 3
    want[2] = want[0] = want[1] = 1
    assert counts == want


@pytest.mark.parametrize("bad", [-1, 20])
def test_a_child_of_a_missing_last_page_reads_as_its_parent(bad):
    """NaN, and not what a former owner left in a free page."""
    g, heads, dim = gen(3), 2, 64
    kc, ks = kv_plain.empty_cache("int8", 20, 8, heads, dim)
    vc, vs = kv_plain.empty_cache("int8", 20, 8, heads, dim)
    every = torch.arange(160)
    for codes, scales in ((kc, ks), (vc, vs)):
        kv_plain.put(codes, scales, "int8", every // 8, every % 8, torch.randn(160, heads, dim, generator=g))
    pool = _pool([[3, 7, bad], []], [21, 0], 20, 4)
    caches = [t.to(DEV) for t in (kc, vc, ks, vs)]
    src, dst = custom_ops.kv_cache_fork(*pool, _i32([0]), _i32([1]), 8)
    custom_ops.kv_cache_copy_pages(caches, src, dst)
    query = torch.randn(2, 4, dim, generator=g).to(DEV)
    out, lse = custom_ops.kv_cache_attention(query, *caches, pool[0], pool[1], return_lse=True)
    assert torch.isnan(out).all() and torch.isnan(lse).all()
    out = custom_ops.kv_cache_attention(query, *caches, pool[0], _i32([16, 16]))  # the whole pages are shared
    assert torch.isfinite(out).all()
    # tokens behind it: no slots inside the missing page, new pages behind it
    slots, starts = custom_ops.kv_cache_extend(*pool, _i32([1]), _i32([0, 5]), 5, 8)
    assert starts.tolist() == [21] and slots.tolist() == [-1, -1, -1, 0, 1]
    assert pool[0].tolist() == [[3, 7, bad, -1], [3, 7, -1, 0]]


@pytest.mark.parametrize("columns", [3, 4])
@pytest.mark.parametrize("behind", [0, 5000])  # in one launch, in two
def test_lengths_end_at_32_bits(behind, columns):
    """A sequence whose new length is no int32 stays as it was, though its row and the pool have room."""
    say(f"lengths up to 2^31, rows of {columns}, {behind} tokens behind")
    most, page = (1 << 31) - 1, 1 << 30
    pool = _pool([[1, 4], [], []], [most - 1, 0, 0], 6, columns)
    before = [t.tolist() for t in pool]
    for add in (2, 4, most):
        slots, starts = custom_ops.kv_cache_extend(*pool, _i32([0]), _i32([0, add]), 4 + behind, page)
        assert starts.tolist() == [-1] and (slots == -1).all()
        assert [t.tolist() for t in pool] == before
    slots, starts = custom_ops.kv_cache_extend(*pool, _i32([0, 1]), _i32([0, 4, 6]), 6 + behind, page)
    assert starts.tolist() == [-1, 0] and slots.tolist() == [-1] * 4 + [0, 1] + [-1] * behind
    slots, starts = custom_ops.kv_cache_extend(*pool, _i32([0]), _i32([0, 1]), 1 + behind, page)
    assert starts.tolist() == [most - 1] and slots.tolist() == [4 * page + page - 2] + [-1] * behind
    none = [-1] * columns
    assert pool[0].tolist() == [[1, 4, *none[2:]], [0, *none[1:]], none]
    assert pool[1].tolist() == [most, 2, 0] and pool[2].tolist() == [1, 1, 0, 0, 1, 0]
    custom_ops.kv_cache_free(*pool, _i32([0, 1]), page)
    assert pool[0].tolist() == [none] * 3 and pool[1].tolist() == [0, 0, 0] and pool[2].tolist() == [0] * 6
