"""The page operators of the cache on the GPU against the pool as lists: copies of every size and
alignment, forks, extensions, ends of sequences and compactions, with requests that do not fit, repeated
ones, pools without a free page, and a serving loop of them with the cache's other operators."""

import pytest
import torch

import kv_plain
import mcoplib_amd._C  # noqa: F401
from gpu_util import DEV, gen, say
from mcoplib import custom_ops
from mcoplib_amd import _C

pytestmark = pytest.mark.gpu


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


class Both:
    """A pool on the device beside one of lists."""

    def __init__(self, pages, rows, columns, page, lens=(), seed=0, wide=0):
        g = gen(seed + pages + rows)
        self.page = page
        held = [-(-n // page) for n in lens]
        order = torch.randperm(pages, generator=g).to(torch.int32)
        table = torch.full((rows, columns), -1, dtype=torch.int32)
        at = 0
        for s, k in enumerate(held):
            table[s, :k] = order[at:at + k]
            at += k
        assert at <= pages
        counts = torch.zeros(pages, dtype=torch.int32)
        counts[order[:at].long()] = 1
        length = torch.zeros(rows, dtype=torch.int32)
        length[:len(lens)] = torch.tensor(lens, dtype=torch.int32)
        base = torch.full((rows, columns + wide), -9, dtype=torch.int32, device=DEV)
        self.base, self.wide = base, wide
        self.table = base[:, wide:]
        self.table.copy_(table)
        self.lens, self.counts = length.to(DEV), counts.to(DEV)
        self.plain = kv_plain.PagePool(table, length, counts, page)

    @property
    def pool(self):
        return self.table, self.lens, self.counts

    def same(self, what):
        assert self.table.tolist() == self.plain.table, f"{what}: table"
        assert self.lens.tolist() == self.plain.lens, f"{what}: lengths"
        assert self.counts.tolist() == self.plain.counts, f"{what}: counts"
        assert (self.base[:, :self.wide] == -9).all()

    def fork(self, parents, children):
        src, dst = custom_ops.kv_cache_fork(*self.pool, _i32(parents), _i32(children), self.page)
        assert [src.tolist(), dst.tolist()] == list(self.plain.fork(parents, children))
        self.same("fork")
        return src, dst

    def extend(self, sequences, add, behind=0):
        cu = [0]
        for a in add:
            cu.append(cu[-1] + a)
        slots, starts = custom_ops.kv_cache_extend(*self.pool, _i32(sequences), _i32(cu),
                                                   cu[-1] + behind, self.page)
        want = self.plain.extend(sequences, cu, cu[-1] + behind)
        assert [slots.tolist(), starts.tolist()] == list(want)
        self.same("extend")
        return slots, starts

    def free(self, sequences):
        custom_ops.kv_cache_free(*self.pool, _i32(sequences), self.page)
        self.plain.free(sequences)
        self.same("free")

    def compact(self):
        src, dst, used = custom_ops.kv_cache_compact(self.table, self.counts)
        assert [src.tolist(), dst.tolist(), used.tolist()] == list(self.plain.compact())
        self.same("compact")
        return src, dst, used


# ------------------------------------------------------------------------------------------ copies


@pytest.mark.parametrize("shape,dtype", [
    ((16, 8, 128), torch.int8), ((16, 8), torch.float32), ((1,), torch.uint8), ((3, 5), torch.uint8),
    ((17,), torch.int8), ((7, 5, 61), torch.float8_e4m3fn), ((64, 16, 256), torch.uint8),
    ((1024, 16), torch.uint8), ((16385,), torch.uint8), ((), torch.float32), ((15,), torch.uint8)])
@pytest.mark.parametrize("pages,pairs", [(2, 1), (9, 4), (130, 65), (40, 0)])
def test_copies_of_every_size(pages, pairs, shape, dtype):
    say(f"copy {pairs} of {pages} pages of {shape} {dtype}")
    g = gen(pages)
    raw = torch.randint(0, 256, (pages, *shape, dtype.itemsize), generator=g, dtype=torch.uint8)
    t = raw.flatten(-2).view(dtype) if shape else raw.view(dtype)[:, 0]
    order = torch.randperm(pages, generator=g)
    src, dst = order[:pairs].clone(), order[pairs:2 * pairs].clone()
    want = raw.clone()
    want[dst] = raw[src]
    if pairs > 2:  # padding, a page of its own, and pages that there are not
        src, dst = (torch.cat([torch.tensor(x), y]) for x, y in (
            ([-1, 3, pages, 0, 1, -(1 << 31)], src), ([0, -1, 1, pages + 5, 1, 1], dst)))
    on = t.to(DEV)
    custom_ops.kv_cache_copy_pages([on], _i32(src.tolist()), _i32(dst.tolist()))
    got = on.cpu()
    assert torch.equal(got.reshape(pages, -1).contiguous().view(torch.uint8), want.reshape(pages, -1))


def test_many_tensors_of_many_layouts():
    """More tensors than a launch takes; pages in strides, heads before tokens, at odd addresses."""
    g = gen(1)
    pages, pairs = 31, 12
    tensors = []
    for i in range(150):
        page, heads, width = 1 + i % 9, 1 + i % 4, 5 + i % 40
        whole = torch.randint(0, 256, (pages, 2, page * heads * width + 3), generator=g,
                              dtype=torch.uint8, device="cpu").to(DEV)
        t = whole[:, 1, 1:1 + page * heads * width].unflatten(1, (heads, page, width))
        tensors.append(t.transpose(1, 2) if i % 2 else t)
    before = [t.cpu().clone() for t in tensors]
    bases = [t.cpu()._base if t.cpu()._base is not None else t.cpu() for t in tensors]
    del bases
    order = torch.randperm(pages, generator=g)
    src, dst = order[:pairs], order[pairs:2 * pairs]
    torch.ops._C.kv_cache_copy_pages(tensors, _i32(src.tolist()), _i32(dst.tolist()))
    for t, old in zip(tensors, before):
        want = old.clone()
        want[dst] = old[src]
        assert torch.equal(t.cpu(), want)


def test_what_lies_between_pages_stays():
    whole = torch.full((6, 3, 50), 7, dtype=torch.uint8, device=DEV)
    t = whole[:, 1, 2:49]
    t.copy_(torch.arange(6, device=DEV)[:, None].expand(6, 47))
    _C.kv_cache_copy_pages([t], _i32([0, 1]), _i32([5, 4]))
    assert (t[5] == 0).all() and (t[4] == 1).all()
    t.fill_(7)
    assert (whole == 7).all()


def test_copies_past_32_bits():
    t = torch.empty(33, 1 << 27, dtype=torch.uint8, device=DEV)  # 4.4e9 bytes
    t[0].fill_(3), t[32].fill_(4), t[31].fill_(5)
    custom_ops.kv_cache_copy_pages([t], _i32([32, 0]), _i32([1, 31]))
    assert (t[1] == 4).all() and (t[31] == 3).all() and (t[32] == 4).all()


def test_no_tensors_no_pairs_no_bytes():
    none = _i32([])
    t = torch.arange(4, device=DEV)
    custom_ops.kv_cache_copy_pages([], _i32([0]), _i32([1]))
    custom_ops.kv_cache_copy_pages([t], none, none)
    custom_ops.kv_cache_copy_pages([torch.empty(4, 0, device=DEV), t], _i32([0]), _i32([3]))
    assert t.tolist() == [0, 1, 2, 0]


# ------------------------------------------------------------------------------------ the pool


@pytest.mark.parametrize("page", [1, 7, 16])
@pytest.mark.parametrize("wide", [0, 3])
def test_forks(page, wide):
    lens = [0, 1, page, page + 1, 5 * page, 5 * page + page // 2]
    both = Both(100, 30, 8, page, lens, wide=wide)
    both.fork([3], [10])
    both.fork([5, 5, 0, 4, 3, 1], [11, 20, 12, 19, 13, 14])
    both.fork([11, 13], [15, 16])  # forks of forks
    both.fork([], [])


def test_forks_that_are_no_forks():
    both = Both(50, 12, 8, 16, [40, 16, 20])
    both.fork([-1, 0, 12, 0, 1 << 30, 2], [5, -1, 6, 12, 7, 8])
    both.lens[2] = 8 * 16 + 1  # longer than its row
    both.plain.lens[2] = 8 * 16 + 1
    both.fork([2, 0], [9, 10])
    both.lens[2] = both.plain.lens[2] = -3
    both.fork([2, 0], [9, 11])


def test_forks_of_an_empty_pool_of_pages():
    """Some forks get the last free pages, whole ones need none."""
    both = Both(8, 12, 8, 16, [40, 16, 20])  # 3 + 1 + 2 of 8
    both.fork([0, 2, 0, 1, 2], [3, 4, 5, 6, 7])
    none = Both(0, 4, 0, 16)
    none.fork([0, 1], [2, 3])


@pytest.mark.parametrize("page", [1, 7, 16])
def test_extensions(page):
    both = Both(300, 20, 12, page, [0, 1, page, page + 1, 3 * page], wide=2)
    both.extend([0, 1, 2, 3, 4], [1, 1, 1, 1, 1])
    both.extend([4, 3, 9, 0], [0, 2 * page, 5 * page + 1, page], behind=7)
    both.extend([5], [12 * page])
    both.extend([], [], behind=3)
    both.extend([6], [12 * page + 1])  # more than its row
    both.extend([6, 7], [0, 0])


def test_extensions_that_do_not_fit():
    both = Both(10, 8, 12, 4, [4, 6, 1])  # 1 + 2 + 1 of 10
    both.extend([0, 1, 2, 3, 4], [4, 2, 40, 1, 0])  # the third takes more than there are
    both.extend([-1, 8, 0, 1 << 30], [3, 2, 2, 1])
    both.extend([5, 6], [24, 4])  # exactly what is left, then nothing
    both.extend([6, 5], [1, 0])


def test_decreasing_token_counts_grow_nothing():
    both = Both(10, 8, 12, 4, [4, 6, 1])
    cu = [0, 3, 1, 4]
    slots, starts = custom_ops.kv_cache_extend(*both.pool, _i32([0, 1, 2]), _i32(cu), 4, 4)
    assert starts.tolist()[1] == -1
    assert both.lens.tolist()[:3] == [7, 6, 4]


# Few requests of short rows are written by the workgroup that takes their pages, in parts of a wave, waves or
# several of them; more or longer ones by a launch of their own.
@pytest.mark.parametrize("forks,columns", [(1, 5), (1, 4096), (1, 4097), (2, 2048), (2, 2049), (3, 1024), (5, 513),
                                           (16, 256), (17, 128), (17, 129), (64, 64), (100, 32), (1000, 4),
                                           (1024, 4), (1024, 5), (1025, 4)])
def test_forks_of_few_and_of_many(forks, columns):
    lens = [columns * 3, columns * 3 - 2, 1, 0]
    both = Both(2 * columns + 1 + forks - forks // 3, 4 + forks, columns, 3, lens)  # some get none
    both.fork([i % 4 for i in range(forks)], [4 + (i * 7 + 3) % forks if forks % 7 else 4 + i
                                              for i in range(forks)])


@pytest.mark.parametrize("sequences,tokens", [(1, 1), (1, 2048), (1, 2049), (2, 1024), (2, 1025), (3, 1025),
                                              (7, 512), (7, 513), (31, 128), (31, 129), (32, 100), (63, 64),
                                              (127, 127), (255, 255), (500, 500), (1023, 1023), (1024, 1024)])
def test_extensions_of_few_and_of_many(sequences, tokens):
    """All tokens in one sequence, then spread over all; other entries of the table lie behind."""
    both = Both(3 * sequences + tokens // 3, sequences + 2, tokens // 2 + 3, 4, [i % 6 for i in range(sequences)])
    order = [(i * 5 + 1) % sequences for i in range(sequences)] if sequences % 5 else list(range(sequences))
    both.extend(order, [tokens if i == sequences // 2 else 0 for i in range(sequences)])
    both.extend(order, [tokens // sequences] * sequences, behind=3)
    both.extend(order, [1] * sequences)


@pytest.mark.parametrize("page", [1, 16])
def test_ends_of_sequences(page):
    both = Both(100, 12, 8, page, [5 * page, 1, 0, 3 * page + 1, 8 * page])
    both.fork([0, 3], [6, 7])
    both.free([3, 2, -1, 12, 11])
    both.free([7, 0, 7, 7])  # the same one again gives back nothing
    both.free([6, 1, 4])
    assert both.counts.tolist() == [0] * 100
    both.free([])


def test_a_length_past_its_row_gives_back_nothing():
    both = Both(20, 4, 3, 4, [12, 4])
    both.lens[0] = both.plain.lens[0] = 13
    both.free([0, 1])


@pytest.mark.parametrize("pages", [1, 2, 3, 7, 64, 1000, 4096, 4097, 20000])
@pytest.mark.parametrize("share", [0.0, 0.1, 0.5, 0.97, 1.0])
def test_compactions(share, pages):
    say(f"compact {pages} pages, {share} in use")
    used = int(pages * share)
    columns = max(1, used // 3)
    both = Both(pages, 7, columns, 1, [min(columns, used // 3 + 0)] * 3 if used >= 3 else [], seed=pages)
    for c in range(0, used // 3, 2):  # counts of more than one, and a row of stale places
        page = int(both.table[0, c])
        both.counts[page] += 3
        both.plain.counts[page] += 3
        both.table[5, c] = page
        both.plain.table[5][c] = page
    both.compact()
    src, dst, used_now = both.compact()  # nothing is left to move
    assert (src == -1).all() and (dst == -1).all()


def test_compaction_leaves_what_is_no_page():
    both = Both(16, 3, 4, 1, [3])
    both.table[2] = _i32([-1, 16, -(1 << 31), 1 << 30])
    both.plain.table[2] = [-1, 16, -(1 << 31), 1 << 30]
    both.counts[:] = _i32([0] * 12 + [-4, 1, 0, 2])
    both.plain.counts = both.counts.tolist()
    both.table[0, :3] = _i32([13, 15, 15])
    both.plain.table[0][:3] = [13, 15, 15]
    both.compact()


def test_large_pools():
    """More requests than a workgroup has threads, free pages far behind, long rows."""
    lens = [int(x) for x in torch.randint(0, 60, (1500,), generator=gen(3))]
    both = Both(70000, 4000, 40, 4, lens)
    both.extend(list(range(1500)), [int(x) for x in torch.randint(0, 30, (1500,), generator=gen(4))])
    parents = [int(x) for x in torch.randint(0, 1500, (2000,), generator=gen(5))]
    both.fork(parents, list(range(1500, 3500)))
    both.free(list(range(0, 3000, 2)))
    both.compact()
    far = Both(100000, 3, 100000, 1, [99990])
    far.extend([1], [10])
    far.extend([1, 0], [1, 0])


def test_other_streams_and_graphs():
    """A step captured and replayed among other work gives what it gives eagerly, each time."""
    both = Both(400, 40, 20, 16, [int(x) for x in torch.randint(1, 200, (10,), generator=gen(7))])
    parents, children = _i32([i % 10 for i in range(20)]), _i32(list(range(12, 32)))
    cu = _i32([i * 3 for i in range(21)])
    cache = torch.randint(0, 256, (400, 16, 2, 8), dtype=torch.uint8, device=DEV)

    def step():
        src, dst = custom_ops.kv_cache_fork(*both.pool, parents, children, 16)
        custom_ops.kv_cache_copy_pages([cache], src, dst)
        slots, starts = custom_ops.kv_cache_extend(*both.pool, children, cu, 60, 16)
        table = both.table.clone()
        custom_ops.kv_cache_free(*both.pool, children, 16)
        return src, dst, slots, starts, table

    want = [t.clone() for t in step()]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, again))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for _ in range(4):
        for t in outs:
            t.fill_(77)
        junk = torch.full((1 << 20,), 5, device=DEV)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, outs))
        del junk
    both.same("after")


# -------------------------------------------------------------------------------- a serving loop


@pytest.mark.parametrize("kind", ["int8", "fp8", "mxfp4"])
@pytest.mark.parametrize("page", [16, 5])
def test_a_serving_loop(kind, page):
    """Prompts, forks, decode steps, ends and a compaction, with the attention of every step against the
    tokens that each sequence was given."""
    heads, group, dim, dtype = 2, 4, 64, torch.bfloat16
    g = gen(11)
    both = Both(200, 12, 40, page, [])
    sides = [kv_plain.empty_cache(kind, 200, page, heads, dim) for _ in range(2)]
    kc, vc = sides[0][0].to(DEV), sides[1][0].to(DEV)
    ks, vs = sides[0][1].to(DEV), sides[1][1].to(DEV)
    texts = {}  # the keys and values of each sequence

    def grow(sequences, add):
        slots, _ = both.extend(sequences, add)
        k, v = (torch.randn(sum(add), heads, dim, generator=g).to(dtype) for _ in range(2))
        custom_ops.kv_cache_write_quant(k.to(DEV), v.to(DEV), kc, vc, ks, vs, slots)
        at = 0
        for s, n in zip(sequences, add):
            old = texts.get(s, (k[:0], v[:0]))
            texts[s] = (torch.cat([old[0], k[at:at + n]]), torch.cat([old[1], v[at:at + n]]))
            at += n

    def attend(what):
        q = torch.randn(12, heads * group, dim, generator=g).to(dtype)
        got, lse = custom_ops.kv_cache_attention(q.to(DEV), kc, vc, ks, vs, both.table, both.lens,
                                                 return_lse=True)
        # a cache of its own for each sequence, one page long
        n = max(1, *(t[0].shape[0] for t in texts.values()))
        own = [kv_plain.empty_cache(kind, 12, n, heads, dim) for _ in range(2)]
        for s, sides in texts.items():
            for (codes, scales), x in zip(own, sides):
                at = torch.full((x.shape[0],), s)
                kv_plain.put(codes, scales, kind, at, torch.arange(x.shape[0]), x)
        lens = torch.tensor([texts[s][0].shape[0] if s in texts else 0 for s in range(12)])
        table = torch.arange(12, dtype=torch.int32)[:, None]
        o, z, ob, zb = kv_plain.attention(q, own[0][0], own[1][0], own[0][1], own[1][1], kind, table, lens,
                                          dim ** -0.5)
        kv_plain.near(got, o, ob, f"{what} out")
        kv_plain.near(lse, z, zb, f"{what} lse")
        return q, got

    grow([0, 1, 2], [37, 1, 64])
    attend("prompts")
    src, dst = both.fork([0, 0, 2], [3, 4, 5])
    custom_ops.kv_cache_copy_pages([kc, vc, ks, vs], src, dst)
    for parent, child in ((0, 3), (0, 4), (2, 5)):
        texts[child] = texts[parent]
    attend("forks")
    for step in range(3):
        grow([0, 1, 2, 3, 4, 5], [1, 2, 1, 1, 1, 1])
        attend(f"step {step}")
    both.free([0, 2])
    del texts[0], texts[2]
    grow([7, 3], [20, 1])
    q, before = attend("ends")
    src, dst, _ = both.compact()
    custom_ops.kv_cache_copy_pages([kc, vc, ks, vs], src, dst)
    after = custom_ops.kv_cache_attention(q.to(DEV), kc, vc, ks, vs, both.table, both.lens)
    assert torch.equal(after, before)
    attend("compacted")
