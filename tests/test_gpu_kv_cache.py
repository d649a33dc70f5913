"""The quantized paged key/value cache on the GPU: codes and scales bit for bit against a plain
statement, over formats, types, head sizes, page sizes and layouts; what a write or a read must leave
alone; pages that the table does not have."""

import math

import pytest
import torch

import mcoplib_amd._C  # noqa: F401
import mx_plain
from gpu_util import DEV, randn, say
from mcoplib import custom_ops

pytestmark = pytest.mark.gpu

KINDS = ["int8", "fp8", "mxfp4"]
CODES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn, "mxfp4": torch.uint8}
FILL = 0x35  # what untouched bytes hold


def _new_cache(kind, pages, page, heads, dim, layout="plain"):
    """(codes, scales) of one side, filled with FILL, on the device."""
    width = dim // 2 if kind == "mxfp4" else dim
    tail = (dim // 32,) if kind == "mxfp4" else ()
    per = 1 if kind == "mxfp4" else 4

    def make(last, size):
        if layout == "heads_first":  # [pages, heads, page, ...] seen as [pages, page, heads, ...]
            t = torch.full((pages, heads, page, last * size), FILL, dtype=torch.uint8, device=DEV)
            return t.transpose(1, 2)
        if layout == "interleaved":  # one of two sides of every page, with a gap after every head
            t = torch.full((pages, 2, page, heads, (last + 3) * size), FILL, dtype=torch.uint8,
                           device=DEV)
            return t[:, 1, :, :, :last * size]
        return torch.full((pages, page, heads, last * size), FILL, dtype=torch.uint8, device=DEV)

    codes = make(width, 1).view(CODES[kind])
    if kind == "mxfp4":
        return codes, make(tail[0], 1)
    return codes, make(1, per).view(torch.float32)[..., 0]


def _bytes(t):
    """The bytes of a cache tensor, one row a slot, on the CPU."""
    t = t.cpu()
    t = t.view(torch.uint8) if t.element_size() == 1 else t.contiguous()
    return t.reshape(t.shape[0] * t.shape[1], *t.shape[2:])


def _check_write(kind, dtype, T, heads, dk, dv, page, layout="plain", fused=False, slots=None,
                 special=False):
    pages = -(-T // page) + 3
    if fused:
        qkv = randn((T, 3 + heads * (dk + dv)), T + dk, dtype, scale=2.0)
        k = qkv[:, 3:3 + heads * dk].unflatten(1, (heads, dk))
        v = qkv[:, 3 + heads * dk:].unflatten(1, (heads, dv))
        on = qkv.to(DEV)
        kd = on[:, 3:3 + heads * dk].unflatten(1, (heads, dk))
        vd = on[:, 3 + heads * dk:].unflatten(1, (heads, dv))
    else:
        k, v = randn((T, heads, dk), T + dk, dtype, scale=2.0), randn((T, heads, dv), 1, dtype)
        if special:
            special(k), special(v)
        kd, vd = k.to(DEV), v.to(DEV)
    if slots is None:
        slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(T))[:T]
    kc, ks = _new_cache(kind, pages, page, heads, dk, layout)
    vc, vs = _new_cache(kind, pages, page, heads, dv, layout)
    custom_ops.kv_cache_write_quant(kd, vd, kc, vc, ks, vs, slots.to(DEV))
    for x, codes, scales in ((k, kc, ks), (v, vc, vs)):
        q, s = mx_plain.vector_codes(x, kind)
        want_q, want_s = _bytes(_fresh(codes)), _bytes(_fresh(scales))
        for t in range(slots.numel()):
            if 0 <= int(slots[t]) < pages * page:
                want_q[int(slots[t])] = q[t].view(torch.uint8)
                want_s[int(slots[t])] = s[t]
        assert mx_plain.same(_bytes(scales), want_s), (kind, dtype, "scales")
        assert torch.equal(_bytes(codes), want_q), (kind, dtype, "codes")
    return (kd, vd), (kc, vc, ks, vs), slots


def _fresh(t):
    f = torch.full((t.numel() * t.element_size(),), FILL, dtype=torch.uint8)
    return f.view(t.dtype).view(t.shape)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 96), (192, 128), (576, 512), (1024, 32),
                                   (80, 80), (61, 7), (1, 513), (256, 1000)])
def test_write(dk, dv, dtype, kind):
    if kind == "mxfp4" and (dk % 32 or dv % 32):
        pytest.skip("4-bit vectors are whole blocks of 32")
    say(f"kv write {kind} {dtype} {dk}/{dv}")
    _check_write(kind, dtype, 37, 3, dk, dv, 16)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("layout", ["heads_first", "interleaved"])
@pytest.mark.parametrize("T,heads,page", [(1, 8, 16), (300, 5, 7), (64, 1, 1), (1000, 2, 64)])
def test_write_layouts(T, heads, page, layout, kind):
    say(f"kv write {kind} {layout} {T} tokens {heads} heads pages of {page}")
    _check_write(kind, torch.bfloat16, T, heads, 96, 64, page, layout, fused=True)
    _check_write(kind, torch.bfloat16, T, heads, 128, 128, page, layout)


@pytest.mark.parametrize("kind", KINDS)
def test_padding_and_slots_past_the_cache(kind):
    """Negative slots, slots past the cache (also past 32 bits) and tokens behind the slots write
    nothing."""
    T, page = 40, 8
    slots = torch.randperm(8 * page, generator=torch.Generator().manual_seed(3))[:T - 5]
    slots[::4], slots[1], slots[2], slots[3] = -1, 8 * page, 1 << 32, -(1 << 40)
    _check_write(kind, torch.bfloat16, T, 2, 64, 64, page, slots=slots)
    none = torch.empty(0, dtype=torch.int64)
    _check_write(kind, torch.bfloat16, T, 2, 64, 64, page, slots=none)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_special_vectors(kind, dtype):
    def special(x):
        x[0] = 0.0
        x[1, 0, 3], x[2, 0, 5] = math.nan, math.inf
        x[3] = torch.finfo(dtype).tiny * 3
        x[4] = torch.finfo(dtype).max / 2
        x[5, 0] = torch.arange(x.shape[-1]) / 8 - 2
        x[6] = -0.0
        x[7] *= 1e-38

    say(f"kv special vectors {kind} {dtype}")
    _check_write(kind, dtype, 16, 2, 64, 32, 16, special=special)


def _check_read(kind, dtype, lengths, starts, heads, dk, dv, page, layout="plain", behind=3,
                width=None):
    """Sequences in pages of random order, read into tensors with rows behind the last sequence."""
    g = torch.Generator().manual_seed(sum(lengths) + dk)
    ends = [n + (s or 0) for n, s in zip(lengths, starts or [0] * len(lengths))]
    held = [-(-e // page) for e in ends]
    pages = sum(held) + 2
    order = torch.randperm(pages, generator=g).to(torch.int32)
    table = torch.full((len(lengths), (width or max(1, max(held))) + 2), -7, dtype=torch.int32)
    at = 0
    for s, n in enumerate(held):
        table[s, :n] = order[at:at + n]
        at += n
    cu = torch.tensor([0] + lengths).cumsum(0).to(torch.int32)
    total, rows = int(cu[-1]), int(cu[-1]) + behind
    outs, caches, wants = [], [], []
    for dim, seed in ((dk, 1), (dv, 2)):
        codes, scales = _new_cache(kind, pages, page, heads, dim, layout)
        q, s = mx_plain.vector_codes(
            torch.randn(pages, page, heads, dim, generator=g, dtype=torch.float32), kind)
        codes.copy_(q.to(DEV)) if kind != "fp8" else codes.view(torch.uint8).copy_(
            q.view(torch.uint8).to(DEV))
        scales.copy_(s.to(DEV))
        caches.append((codes, scales))
        v = mx_plain.vector_values(q, s, kind, dtype)
        want = torch.full((rows, heads, dim), 5.0, dtype=dtype)
        t = 0
        for i, n in enumerate(lengths):
            for p in range(n):
                p += starts[i] if starts else 0
                want[t] = v[int(table[i, p // page]), p % page]
                t += 1
        wants.append(want)
        outs.append(torch.full((rows, heads, dim), 5.0, dtype=dtype, device=DEV))
    (kc, ks), (vc, vs) = caches
    sd = torch.tensor(starts, dtype=torch.int32, device=DEV) if starts else None
    td = table.to(DEV)[:, :table.shape[1] - 2] if width is None else table.to(DEV)
    torch.ops._C.kv_cache_read_dequant(outs[0], outs[1], kc, vc, ks, vs, td, cu.to(DEV), sd)
    for got, want in zip(outs, wants):
        assert mx_plain.same(got, want)
    if total:
        k, v = custom_ops.kv_cache_read_dequant(kc, vc, ks, vs, td, cu.to(DEV), total, dtype, sd)
        assert mx_plain.same(k, wants[0][:total]) and mx_plain.same(v, wants[1][:total])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("dk,dv", [(128, 128), (192, 64), (576, 512), (1024, 32), (80, 80), (61, 7),
                                   (1, 513)])
def test_read(dk, dv, dtype, kind):
    if kind == "mxfp4" and (dk % 32 or dv % 32):
        pytest.skip("4-bit vectors are whole blocks of 32")
    say(f"kv read {kind} {dtype} {dk}/{dv}")
    _check_read(kind, dtype, [17, 1, 30], None, 3, dk, dv, 16)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("layout", ["plain", "heads_first", "interleaved"])
@pytest.mark.parametrize("lengths,starts,page", [
    ([1], None, 16), ([0], None, 16), ([0, 0, 5, 0, 1, 0], None, 4), ([33, 2], [0, 31], 16),
    ([100, 0, 1, 250], [7, 3, 0, 64], 7), ([3] * 150, [1] * 150, 2), ([0] * 200 + [9], None, 1),
    ([500], [1], 64)])
def test_read_sequences(lengths, starts, page, layout, kind):
    say(f"kv read {kind} {layout} {len(lengths)} sequences {sum(lengths)} tokens pages of {page}")
    _check_read(kind, torch.bfloat16, lengths, starts, 2, 64, 96, page, layout)


def test_pages_that_the_table_does_not_have_read_as_nan():
    """A column past the table, a page below 0 or past the cache: NaN, and nothing else changes."""
    page, heads, dim = 4, 2, 64
    for kind in KINDS:
        codes, scales = _new_cache(kind, 3, page, heads, dim)
        q, s = mx_plain.vector_codes(randn((3, page, heads, dim), 1, torch.float32), kind)
        codes.view(torch.uint8).copy_(q.view(torch.uint8).to(DEV))
        scales.copy_(s.to(DEV))
        v = mx_plain.vector_values(q, s, kind, torch.bfloat16)
        table = torch.tensor([[2, -1], [3, 0], [1, 1 << 30]], dtype=torch.int32, device=DEV)
        cu = torch.tensor([0, 9, 14, 22], dtype=torch.int32, device=DEV)
        starts = torch.tensor([0, 2, -3], dtype=torch.int32, device=DEV)
        key, value = custom_ops.kv_cache_read_dequant(codes, codes, scales, scales, table, cu, 22,
                                                      torch.bfloat16, starts)
        want = torch.full((22, heads, dim), math.nan, dtype=torch.bfloat16)
        want[0:4] = v[2]  # then page -1, then past the table
        want[11:14] = v[0, 0:3]  # positions 2, 3 are on page 3 of 3, 4..6 on page 0
        want[17:21] = v[1]  # positions -3..-1, page 1, then page 2^30
        assert mx_plain.same(key, want) and mx_plain.same(value, want), kind
        none = torch.empty(0, page, heads, codes.shape[-1], dtype=codes.dtype, device=DEV)
        no_scales = scales[:0]
        key, _ = custom_ops.kv_cache_read_dequant(none, none, no_scales, no_scales, table, cu, 22,
                                                  torch.bfloat16, starts)
        assert bool(torch.isnan(key).all()), kind


@pytest.mark.parametrize("kind", KINDS)
def test_a_cache_past_32_bit_offsets(kind):
    """Slots whose bytes lie past 2^32 (a cache of 5 GiB a side) are written and read."""
    heads, dim, page = 8, 128, 64
    width = dim // 2 if kind == "mxfp4" else dim
    pages = 5 * (1 << 30) // (heads * width * page)
    say(f"kv past 32-bit offsets {kind}: {pages} pages")
    codes = torch.zeros(pages, page, heads, width, dtype=CODES[kind], device=DEV)
    scales = (torch.zeros(pages, page, heads, 4, dtype=torch.uint8, device=DEV) if kind == "mxfp4"
              else torch.zeros(pages, page, heads, device=DEV))
    T = 70
    k = randn((T, heads, dim), 1, torch.bfloat16)
    slots = torch.arange(T) + (pages - 2) * page
    kd = k.to(DEV)
    custom_ops.kv_cache_write_quant(kd, kd, codes, codes.clone(), scales, scales.clone(),
                                    slots.to(DEV))
    q, s = mx_plain.vector_codes(k, kind)
    flat = codes.view(torch.uint8).flatten(0, 1)
    assert torch.equal(flat[slots[0]:slots[0] + T].cpu(), q.view(torch.uint8))
    assert int(flat[:1 << 20].sum()) == 0
    table = torch.tensor([[pages - 2, pages - 1]], dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, T], dtype=torch.int32, device=DEV)
    key, _ = custom_ops.kv_cache_read_dequant(codes, codes, scales, scales, table, cu, T,
                                              torch.bfloat16)
    assert mx_plain.same(key, mx_plain.vector_values(q, s, kind, torch.bfloat16))


# Tokens enough for waves of several, with a last wave that is not full; the sides differ in how many
# waves a token takes.
MANY = [(4101, 8, 128, 128), (2051, 16, 128, 32), (4099, 9, 61, 64), (8195, 1, 576, 512),
        (8193, 3, 1024, 520)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T,heads,dk,dv", MANY)
def test_write_many_tokens(T, heads, dk, dv, kind):
    if kind == "mxfp4" and (dk % 32 or dv % 32):
        pytest.skip("4-bit vectors are whole blocks of 32")
    say(f"kv write {kind} {T} tokens of {heads} x {dk}/{dv}")
    _check_write(kind, torch.bfloat16, T, heads, dk, dv, 16)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,heads,dk,dv", MANY)
def test_read_many_tokens(T, heads, dk, dv, kind, dtype):
    """Sequences of every length from 0 to 6 among long ones, so that a wave's tokens are of several."""
    if kind == "mxfp4" and (dk % 32 or dv % 32):
        pytest.skip("4-bit vectors are whole blocks of 32")
    say(f"kv read {kind} {dtype} {T} tokens of {heads} x {dk}/{dv}")
    lengths = [n % 7 for n in range(150)] + [700, 0, 0, 1]
    lengths.append(T - sum(lengths))
    _check_read(kind, dtype, lengths, [n % 5 for n in range(len(lengths))], heads, dk, dv, 16)
