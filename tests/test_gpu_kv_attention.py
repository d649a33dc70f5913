"""kv_cache_attention on the GPU against a plain statement in 64 bits: formats, types, head layouts, lengths
from none to thousands, pages, windows, layouts and strides; slots that must not be read, pages that the
table does not have, special values; streams, graphs and offsets past 32 bits."""

import math

import pytest
import torch

import kv_plain
import mcoplib_amd._C  # noqa: F401
from gpu_util import DEV, gen, say
from mcoplib import custom_ops
from mcoplib_amd import _C

pytestmark = pytest.mark.gpu

KINDS = ["int8", "fp8", "mxfp4"]
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


class Case:
    """A cache whose slots outside the sequences read as NaN, in pages of random order."""

    def __init__(self, kind, dtype, lens, heads, group, dk, dv, page, layout="plain", window=0, loud=1.0,
                 seed=0, fused=False):
        g = gen(seed + sum(lens) + dk)
        self.kind, self.window, self.page, self.heads = kind, window, page, heads
        self.lens = torch.tensor(lens, dtype=torch.int32)
        held = (self.lens.clamp_min(0) + page - 1) // page
        columns, pages = max(1, int(held.max())), int(held.sum()) + 3
        order = torch.randperm(pages, generator=g).to(torch.int32)
        self.table = torch.full((len(lens), columns), -1, dtype=torch.int32)
        self.table[torch.arange(columns).expand_as(self.table) < held[:, None]] = order[:int(held.sum())]
        self.kc, self.ks = kv_plain.empty_cache(kind, pages, page, heads, dk, layout)
        self.vc, self.vs = kv_plain.empty_cache(kind, pages, page, heads, dv, layout)
        for b, n in enumerate(lens):
            p = torch.arange(max(0, n - window) if window else 0, max(0, n))
            at, off = self.table[b].long()[p // page], p % page
            kv_plain.put(self.kc, self.ks, kind, at, off, torch.randn(len(p), heads, dk, generator=g))
            kv_plain.put(self.vc, self.vs, kind, at, off, torch.randn(len(p), heads, dv, generator=g))
        q = (torch.randn(len(lens), heads * group, dk, generator=g) * loud).to(dtype)
        self.query, self.scale = q, dk ** -0.5
        if fused:  # as slices of a wider row
            wide = torch.zeros(len(lens), heads * group * dk + 5, dtype=dtype)
            wide[:, 3:3 + heads * group * dk] = q.flatten(1)
            self.on_query = wide.to(DEV)[:, 3:3 + heads * group * dk].unflatten(1, (heads * group, dk))
        else:
            self.on_query = q.to(DEV)

    def device(self):
        return [_same_layout(t) for t in (self.kc, self.vc, self.ks, self.vs)] + [
            self.table.to(DEV), self.lens.to(DEV)]

    def want(self):
        return kv_plain.attention(self.query, self.kc, self.vc, self.ks, self.vs, self.kind, self.table,
                                  self.lens, self.scale, self.window)

    def check(self, what=""):
        out, lse = custom_ops.kv_cache_attention(self.on_query, *self.device(), window=self.window,
                                                 return_lse=True)
        assert out.dtype == self.query.dtype and lse.dtype == torch.float32
        self.compare(out, lse, what)
        return out, lse

    def compare(self, out, lse, what=""):
        o, z, ob, zb = self.want()
        kv_plain.near(lse, z, zb, f"{what} lse")
        kv_plain.near(out, o, ob, f"{what} out")


def _same_layout(t):
    """t on the device with its strides (a copy of all that its storage holds)."""
    raw = t.view(torch.uint8) if t.element_size() == 1 else t
    base = torch.empty(0, dtype=raw.dtype).set_(raw.untyped_storage()).to(DEV)
    return base.as_strided(raw.shape, raw.stride(), raw.storage_offset()).view(t.dtype)


SHAPES = [(128, 128), (64, 64), (80, 96), (192, 128), (256, 256), (16, 16), (61, 7), (1, 1), (576, 512),
          (1024, 32), (32, 1000), (96, 160), (40, 200)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dk,dv", SHAPES)
def test_head_sizes(dk, dv, dtype, kind):
    if kind == "mxfp4":
        dk, dv = -(-dk // 32) * 32, -(-dv // 32) * 32
    say(f"attention {kind} {dtype} {dk}/{dv}")
    Case(kind, dtype, [1, 0, 37, 300], 2, 4, dk, dv, 16).check()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("page", [1, 7, 16, 64, 100])
def test_lengths_and_pages(page, kind):
    lens = [1, 0, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 1000]
    say(f"attention {kind} lengths, pages of {page}")
    Case(kind, torch.bfloat16, lens, 2, 3, 64, 96, page).check()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,group", [(1, 1), (8, 1), (1, 16), (1, 17), (5, 3), (2, 40), (4, 8),
                                         (3, 64), (1, 128), (600, 1)])
def test_head_layouts(heads, group, kind):
    say(f"attention {kind} {heads} heads, groups of {group}")
    Case(kind, torch.float16, [5, 200, 0, 64], heads, group, 64, 64, 16).check()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lens", [[5000, 3, 700, 0, 1], [9000], [4097, 4095], [0, 0], [1]])
def test_split_lengths(lens, dtype, kind):
    """Sequences of many chunks beside short ones."""
    say(f"attention {kind} {dtype} lengths {lens}")
    Case(kind, dtype, lens, 2, 8, 128, 128, 16).check()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("sequences", [127, 255, 256, 400])
def test_more_sequences_than_shares(sequences, dtype, kind):
    """On both sides of two sequences a share, some of them cut."""
    say(f"attention {kind} {dtype} {sequences} sequences")
    lens = [(i * 37) % 90 if i % 50 else 400 for i in range(sequences)]
    Case(kind, dtype, lens, 8, 2, 96, 128, 16).check()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 100, 128, 129, 5000])
def test_windows(window, kind):
    """Only the window's positions are read: those before it read as NaN, and have no pages."""
    case = Case(kind, torch.bfloat16, [1, 31, 32, 33, 100, 129, 2000, 0], 2, 4, 64, 64, 16, window=window)
    for b, n in enumerate(case.lens.tolist()):
        case.table[b, :max(0, n - window) // 16] = -1
    say(f"attention {kind} window {window}")
    case.check()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("layout", ["heads_first", "interleaved"])
@pytest.mark.parametrize("dk,dv", [(128, 128), (96, 64), (192, 256)])
def test_layouts(dk, dv, layout, kind):
    say(f"attention {kind} {layout} {dk}/{dv}")
    Case(kind, torch.bfloat16, [200, 3, 130], 3, 4, dk, dv, 16, layout, fused=True).check()


@pytest.mark.parametrize("sequences", [63, 64, 65, 300, 1000])
def test_many_sequences(sequences):
    lens = torch.randint(0, 90, (sequences,), generator=gen(sequences)).tolist()
    lens[sequences // 2] = 700
    say(f"attention of {sequences} sequences")
    Case("int8", torch.bfloat16, lens, 2, 2, 32, 32, 16).check()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_one_position_takes_all(dtype, kind):
    """Logits of some hundreds: weights of one and of nothing."""
    say(f"attention {kind} {dtype} loud queries")
    Case(kind, dtype, [1, 77, 1500], 2, 4, 128, 128, 16, loud=60.0).check()


@pytest.mark.parametrize("kind", KINDS)
def test_missing_pages(kind):
    """A sequence with a position that has no page is NaN, the others are as they were."""
    case = Case(kind, torch.bfloat16, [40, 300, 1000, 20, 64], 2, 4, 64, 64, 16)
    whole, _ = case.check()
    case.table[1, 3] = -1
    case.table[2, 20] = case.kc.shape[0]
    case.table[3, 0] = -(1 << 31)
    out, _ = case.check("missing")
    assert torch.isnan(out[1:4]).all() and torch.equal(out[[0, 4]], whole[[0, 4]])
    case.lens[0], case.lens[4] = case.table.shape[1] * 16 + 1, (1 << 31) - 1  # past the table
    assert torch.isnan(case.check("too long")[0]).all()
    case.lens[:] = torch.tensor([-1, -(1 << 31), 0, 0, -5])  # no positions
    out, lse = case.check("negative")
    assert (out == 0).all() and (lse == -math.inf).all()


def test_a_cache_of_no_pages_and_a_table_of_no_columns():
    q = torch.ones(2, 4, 64, dtype=torch.bfloat16, device=DEV)
    codes = torch.zeros(0, 16, 2, 64, dtype=torch.int8, device=DEV)
    scales = torch.zeros(0, 16, 2, device=DEV)
    lens = torch.tensor([0, 3], dtype=torch.int32, device=DEV)
    for columns in (0, 1):
        table = torch.zeros(2, columns, dtype=torch.int32, device=DEV)
        out, lse = custom_ops.kv_cache_attention(q, codes, codes, scales, scales, table, lens,
                                                 return_lse=True)
        assert (out[0] == 0).all() and (lse[0] == -math.inf).all()
        assert torch.isnan(out[1]).all() and torch.isnan(lse[1]).all()
    none = custom_ops.kv_cache_attention(q[:0], codes, codes, scales, scales, table[:0], lens[:0])
    assert none.shape == (0, 4, 64)


@pytest.mark.parametrize("kind", KINDS)
def test_special_values(kind):
    """NaN and infinities that are read spoil what the formula says and no more: a key the rows of its
    head, a value the elements that it reaches."""
    case = Case(kind, torch.float32, [100, 90, 300], 3, 2, 64, 64, 16)
    page, off = case.table[0].long()[50 // 16], 50 % 16
    if kind == "mxfp4":
        case.ks[page, off, 1, 1] = 255
        case.vs[page, off, 2, 0] = 255
    else:
        case.ks[page, off, 1] = math.nan
        case.vs[page, off, 2] = math.nan
    if kind == "fp8":
        case.vc.view(torch.uint8)[case.table[1].long()[0], 3, 0, 17] = 0x7F
    case.query[2, 3, 5] = math.nan
    case.on_query = case.query.to(DEV)
    out, _ = case.check(kind)
    out = out.cpu()
    assert torch.isnan(out[0, 2:4]).all() and not torch.isnan(out[0, :2]).any()
    assert torch.isnan(out[0, 4:, :32]).all()
    assert bool(torch.isnan(out[0, 4:, 32:]).any()) == (kind != "mxfp4")
    assert torch.isnan(out[2, 3]).all() and not torch.isnan(out[2, 2]).any()
    assert int(torch.isnan(out[1]).sum()) == (2 if kind == "fp8" else 0)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("power", [-60, 40])
def test_far_scales(power, kind):
    """Vectors of very different sizes: a scale of 2^power beside ordinary ones."""
    case = Case(kind, torch.bfloat16, [70, 400], 2, 4, 64, 64, 16)
    p = torch.arange(0, 400, 3)
    at, off = case.table[1].long()[p // 16], p % 16
    kv_plain.put(case.vc, case.vs, kind, at, off,
                 torch.randn(len(p), 2, 64, generator=gen(5)) * 2.0 ** power)
    kv_plain.put(case.kc, case.ks, kind, at, off,
                 torch.randn(len(p), 2, 64, generator=gen(6)) * 2.0 ** min(power, 0))
    say(f"attention {kind} scales of 2^{power}")
    case.check()


def test_values_at_the_ends_of_the_range():
    """Scales near fp32's smallest and largest: weights times scales neither vanish nor overflow alone."""
    for scale in (1e-37, 1e37):
        case = Case("int8", torch.float32, [50, 300], 2, 4, 64, 64, 16)
        case.vs[~torch.isnan(case.vs)] = scale
        case.check(f"scale {scale}")


def test_given_scale_and_outputs_in_place():
    """The _C form: a given scale, a strided result whose gaps stay, and lse."""
    case = Case("fp8", torch.bfloat16, [0, 40, 700], 2, 4, 64, 96, 16)
    case.scale = 0.37
    wide = torch.full((3, 8, 100), 7.0, dtype=torch.bfloat16, device=DEV)
    lse = torch.full((3, 8), 7.0, device=DEV)
    _C.kv_cache_attention(wide[:, :, 2:98], case.on_query, *case.device(), 0.37, 0, lse)
    case.compare(wide[:, :, 2:98], lse)
    assert (wide[:, :, :2] == 7).all() and (wide[:, :, 98:] == 7).all()
    torch.ops._C.kv_cache_attention(wide[:, :, 2:98], case.on_query, *case.device(), 0.37, 0, None)
    case.compare(wide[:, :, 2:98], lse)


def test_table_rows_of_a_wider_table():
    case = Case("int8", torch.bfloat16, [300, 40], 2, 4, 64, 64, 16)
    wide = torch.full((2, 50), -7, dtype=torch.int32)
    wide[:, 5:5 + case.table.shape[1]] = case.table
    args = case.device()
    args[4] = wide.to(DEV)[:, 5:5 + case.table.shape[1]]
    out, lse = custom_ops.kv_cache_attention(case.on_query, *args, return_lse=True)
    case.compare(out, lse)


def test_halves_join_by_their_sums():
    """Attention over a sequence's halves, joined by lse, is attention over the sequence."""
    case = Case("fp8", torch.float32, [512], 2, 4, 128, 128, 16)
    kc, vc, ks, vs, table, _ = case.device()
    half = torch.tensor([256], dtype=torch.int32, device=DEV)
    parts = [custom_ops.kv_cache_attention(case.on_query, kc, vc, ks, vs, t.contiguous(), half,
                                           return_lse=True)
             for t in (table[:, :16], table[:, 16:])]
    top = torch.maximum(parts[0][1], parts[1][1]).double()
    w = [torch.exp(z.double() - top) for _, z in parts]
    out = sum(o.double() * f[..., None] for (o, _), f in zip(parts, w)) / sum(w)[..., None]
    o, z, ob, zb = case.want()
    kv_plain.near((top + sum(w).log()).float(), z, 2 * zb, "joined lse")
    kv_plain.near(out.float(), o, 2 * ob + zb.amax() * ob.new_tensor(8.0), "joined out")


def test_repeats_are_the_same():
    case = Case("int8", torch.bfloat16, [5000, 100, 0, 2000], 4, 8, 128, 128, 16)
    args = case.device()
    first = custom_ops.kv_cache_attention(case.on_query, *args, return_lse=True)
    for _ in range(5):
        again = custom_ops.kv_cache_attention(case.on_query, *args, return_lse=True)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_two_streams_at_once():
    cases = [Case(k, torch.bfloat16, [3000, 50], 2, 8, 128, 128, 16, seed=i)
             for i, k in enumerate(KINDS)]
    args = [c.device() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    outs = [[] for _ in cases]
    for _ in range(10):
        for c, a, s, o in zip(cases, args, streams, outs):
            with torch.cuda.stream(s):
                o.append(custom_ops.kv_cache_attention(c.on_query, *a, return_lse=True))
    torch.cuda.synchronize()
    for c, o in zip(cases, outs):
        for out, lse in o:
            assert torch.equal(out, o[0][0]) and torch.equal(lse, o[0][1])
        c.compare(*o[0])


def test_two_graphs_with_new_lengths():
    """Two captured graphs replayed in turn with lengths and queries changed between, eager calls among
    them."""
    cases = [Case("fp8", torch.bfloat16, [1500, 700], 2, 8, 128, 128, 16, seed=i) for i in range(2)]
    args = [c.device() for c in cases]
    queries = [c.on_query.clone() for c in cases]
    eager = lambda i: custom_ops.kv_cache_attention(queries[i], *args[i], return_lse=True)  # noqa: E731
    eager(0), eager(1)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(eager(i))
        graphs.append(g)
    for step, lens in enumerate([[1500, 700], [1, 0], [1500, 3], [129, 700]]):
        for i in range(2):
            args[i][5].copy_(torch.tensor(lens, dtype=torch.int32))
            queries[i].copy_(cases[i].on_query * (1 + step))
            graphs[i].replay()
        want = [eager(0), eager(1)]
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i][0], want[i][0]) and torch.equal(outs[i][1], want[i][1]), step


def test_offsets_past_32_bits():
    """Pages more than 4 GiB into a cache."""
    pages, page, heads, dim = 4200, 64, 64, 256  # 4.4e9 bytes a side
    case = Case("fp8", torch.bfloat16, [200, 90], heads, 1, dim, dim, page)
    used = case.kc.shape[0]
    shift = pages - used
    big = []
    for t in case.device()[:4]:
        whole = torch.zeros(pages, *t.shape[1:], dtype=t.dtype, device=DEV)
        whole.view(torch.uint8)[shift:] = t.view(torch.uint8)
        big.append(whole)
    assert big[0].numel() > 1 << 32
    table = torch.where(case.table >= 0, case.table + shift, case.table).to(DEV)
    out, lse = custom_ops.kv_cache_attention(case.on_query, *big, table, case.lens.to(DEV),
                                             return_lse=True)
    case.compare(out, lse)
