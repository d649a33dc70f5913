"""kv_cache_attention where its numbers end, on the GPU against the formula in 64 bits: weights whose every bit
shows, queries and 4-bit values next to fp32's largest, lengths next to 2^31."""

import math

import pytest
import torch

import kv_plain
import mcoplib_amd._C  # noqa: F401
import mx_plain
from gpu_util import DEV, gen, say
from mcoplib import custom_ops

pytestmark = pytest.mark.gpu

KINDS = ["int8", "fp8", "mxfp4"]
U = 2.0 ** -24  # half a step of fp32


def exact_codes(x, kind):
    """(codes, scales) of vectors whose elements are codes times a power of two in each block of 32."""
    if kind == "mxfp4":
        most = x.double().unflatten(-1, (-1, 32)).abs().amax(-1)
        byte = torch.where(most > 6, 131, 127)
        size = x.double().abs().unflatten(-1, (-1, 32)) * torch.pow(2.0, 127.0 - byte)[..., None]
        code = (size[..., None] == mx_plain.VALUES).int().argmax(-1) + 8 * (x < 0).unflatten(-1, (-1, 32))
        return mx_plain.pack(code.flatten(-2)), byte.to(torch.uint8)
    return x.to(kv_plain.CODES[kind]), torch.ones(x.shape[:-1])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("dk,dv,page", [(64, 64, 16), (128, 128, 16), (192, 128, 16), (256, 256, 16),
                                        (128, 96, 7), (256, 256, 7), (512, 32, 16)])
@pytest.mark.parametrize("n", [2, 40])
def test_weights_keep_their_bits(n, dk, dv, page, dtype, kind):
    """Two positions of weights 1 and w = 2/3 whose values, 2 and -3 in every element, leave nothing but the
    weights' errors: what w loses of its 24 bits is the result.

    The other positions have values of zero and weights of e^-39, which neither sum sees.  The bound, in u =
    2^-24 of |2| + |-3| w = 4: w's exponent is one product of three fp32 factors (scale, log2 e, their product)
    and a rounding, 2.25 u of 0.59, so 0.9 u of w, and its own 2 u; two products, in three terms each, added
    up in steps of 2 u of the largest, 2: 3 u of 4 at most; w's errors reach half of the 4.
    3 u + 2.9 u / 2 < 5 u; a weight of 17 bits is 2^-19 = 32 u of 4 off.
    The sum of the weights is 5/3, and the result's own rounding is of almost nothing."""
    k, v = torch.zeros(n, 1, dk), torch.zeros(n, 1, dv)
    a, b = n // 2 - 1, n // 2
    k[:, 0, 0] = -96.0
    k[a], k[b, 0, 0] = 0.0, -1.0
    v[a], v[b] = 2.0, -3.0
    pages = -(-n // page)
    kc, ks = kv_plain.empty_cache(kind, pages, page, 1, dk)
    vc, vs = kv_plain.empty_cache(kind, pages, page, 1, dv)
    p = torch.arange(n)
    for codes, scales, x in ((kc, ks, k), (vc, vs, v)):
        q, s = exact_codes(x, kind)
        codes.view(torch.uint8)[p // page, p % page] = q.view(torch.uint8)
        scales[p // page, p % page] = s
        assert torch.equal(kv_plain.vectors(codes, scales, kind, p // page, p % page), x.double())
    query = torch.zeros(1, 2, dk, dtype=dtype)
    query[:, :, 0] = 1.0
    scale = float(torch.tensor(math.log(1.5), dtype=torch.float32))
    say(f"attention {kind} {dtype} {dk}/{dv} pages of {page}: 2 w - 3 w' of {n}")
    out = custom_ops.kv_cache_attention(
        query.to(DEV), kc.to(DEV), vc.to(DEV), ks.to(DEV), vs.to(DEV),
        torch.arange(pages, dtype=torch.int32, device=DEV)[None],
        torch.tensor([n], dtype=torch.int32, device=DEV), scale).cpu().double()
    w = math.exp(-scale)
    want = (2 - 3 * w) / (1 + w)
    off = float((out - want).abs().max()) * (1 + w) / (4 * U)
    print(f"  {off:.2f} u", flush=True)
    assert off <= 5.0 + 2.0 ** -8 * abs(want) / U


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dk,dv,page", [(64, 64, 16), (128, 128, 16), (256, 256, 16), (96, 64, 7),
                                        (512, 32, 16)])
def test_fp32_queries_up_to_the_largest(dk, dv, page, kind):
    """Queries that bf16 rounds to infinity (from 3.39e38 on), of one element, beside keys of tiny scales: no sum
    of products leaves fp32's range, and the logits are ordinary ones."""
    n, g, most = 100, gen(dk), torch.finfo(torch.float32).max
    pages = -(-n // page)
    kc, ks = kv_plain.empty_cache(kind, pages, page, 2, dk, poison=False)
    vc, vs = kv_plain.empty_cache(kind, pages, page, 2, dv)
    p = torch.arange(n)
    k = torch.zeros(n, 2, dk)
    k[..., 5] = torch.randint(-1, 2, (n, 2), generator=g).float()
    kc.view(torch.uint8)[p // page, p % page] = exact_codes(k, kind)[0].view(torch.uint8)
    ks[p // page, p % page] = 4 if kind == "mxfp4" else 1e-37
    kv_plain.put(vc, vs, kind, p // page, p % page, torch.randn(n, 2, dv, generator=g))
    query = torch.zeros(1, 8, dk)
    query[0, :, 5] = torch.tensor([most, -most, most * 0.9985, -1e38, most, 3.39e38, 1.0, 0.0])
    table = torch.arange(pages, dtype=torch.int32)[None]
    lens = torch.tensor([n], dtype=torch.int32)
    scale = float(torch.tensor(0.0625))
    say(f"attention {kind} {dk}/{dv} pages of {page}: queries of 3.4e38")
    out, lse = custom_ops.kv_cache_attention(*(t.to(DEV) for t in (query, kc, vc, ks, vs, table, lens)), scale,
                                             return_lse=True)
    o, z, ob, zb = kv_plain.attention(query, kc, vc, ks, vs, kind, table, lens, scale)
    kv_plain.near(lse, z, zb, "lse")
    kv_plain.near(out, o, ob, "out")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("dk", [64, 512])
def test_infinite_queries_spoil_their_own_row(dk, dtype):
    n, g = 100, gen(dk)
    kc, ks = kv_plain.empty_cache("int8", 7, 16, 1, dk, poison=False)
    vc, vs = kv_plain.empty_cache("int8", 7, 16, 1, 64)
    p = torch.arange(n)
    kc[p // 16, p % 16, 0, 5], ks[p // 16, p % 16] = 1, 0.5
    kv_plain.put(vc, vs, "int8", p // 16, p % 16, torch.randn(n, 1, 64, generator=g))
    query = torch.zeros(1, 4, dk, dtype=dtype)
    query[0, :, 5] = torch.tensor([math.inf, 2.0, -math.inf, -1.0], dtype=dtype)
    table, lens = torch.arange(7, dtype=torch.int32)[None], torch.tensor([n], dtype=torch.int32)
    say(f"attention {dtype} {dk}: infinite queries")
    out, lse = custom_ops.kv_cache_attention(*(t.to(DEV) for t in (query, kc, vc, ks, vs, table, lens)), 1.0,
                                             return_lse=True)
    assert torch.isnan(out[0, 0]).all() and not torch.isfinite(lse[0, 0])
    assert torch.isnan(out[0, 2]).all() or ((out[0, 2] == 0).all() and lse[0, 2] == -math.inf)  # all are -inf
    o, z, ob, zb = kv_plain.attention(query[:, 1::2], kc, vc, ks, vs, "int8", table, lens, 1.0)
    kv_plain.near(lse[:, 1::2], z, zb, "lse")
    kv_plain.near(out[:, 1::2], o, ob, "out")


@pytest.mark.parametrize("window", [3, 40, 100])
@pytest.mark.parametrize("kind,dk,dv", [("int8", 8, 8), ("fp8", 320, 16), ("mxfp4", 32, 288), ("int8", 64, 64),
                                        ("fp8", 61, 64), ("mxfp4", 128, 128), ("int8", 256, 200)])
def test_lengths_up_to_the_largest_int32(kind, dk, dv, window):
    """Windows at the end of sequences whose rows of the table name one page again and again: positions and
    the ends of tiles next to 2^31."""
    page, g = 1 << 16, gen(dk + window)
    lens = torch.tensor([(1 << 31) - 1 - x for x in (0, 1, 30, 31, 32, 33, 64)] + [50], dtype=torch.int32)
    kc, ks = kv_plain.empty_cache(kind, 1, page, 2, dk)
    vc, vs = kv_plain.empty_cache(kind, 1, page, 2, dv)
    off = torch.cat([torch.arange(50), torch.arange(page - 200, page)])
    for codes, scales, d in ((kc, ks, dk), (vc, vs, dv)):
        kv_plain.put(codes, scales, kind, torch.zeros_like(off), off, torch.randn(250, 2, d, generator=g))
    query = torch.randn(len(lens), 6, dk, generator=g)
    table = torch.zeros(len(lens), 1 << 15, dtype=torch.int32)
    say(f"attention {kind} {dk}/{dv}, windows of {window} at 2^31")
    out, lse = custom_ops.kv_cache_attention(*(t.to(DEV) for t in (query, kc, vc, ks, vs, table, lens)), 0.1, window,
                                             return_lse=True)
    o, z, ob, zb = kv_plain.attention(query, kc, vc, ks, vs, kind, table, lens, float(torch.tensor(0.1)), window)
    kv_plain.near(lse, z, zb, "lse")
    kv_plain.near(out, o, ob, "out")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 128), (256, 256), (32, 1024)])
@pytest.mark.parametrize("page", [16, 7])
@pytest.mark.parametrize("late", [False, True])
def test_4bit_values_at_the_end_of_the_range(late, page, dk, dv, dtype):
    """Values next to fp32's largest, in all positions or in the last third only, under logits that rise by
    less than a factor of 2^8 of weight: neither a weight times a value nor their sum leaves fp32's range
    where the result does not."""
    lens, g = [300, 3], gen(dk + page)
    pages = sum(-(-n // page) for n in lens)
    kc, ks = kv_plain.empty_cache("mxfp4", pages, page, 2, dk)
    vc, vs = kv_plain.empty_cache("mxfp4", pages, page, 2, dv)
    table = torch.full((2, -(-300 // page)), -1, dtype=torch.int32)
    table[0], table[1, :-(-3 // page)] = torch.arange(table.shape[1]), pages - 1
    for b, n in enumerate(lens):
        p = torch.arange(n)
        at, off = table[b].long()[p // page], p % page
        k = torch.zeros(n, 2, dk)
        k[..., 0] = (5.0 * p / n)[:, None]
        kv_plain.put(kc, ks, "mxfp4", at, off, k)
        v = 1 + torch.rand(n, 2, dv, generator=g)
        kv_plain.put(vc, vs, "mxfp4", at, off, v)
        vs[at, off] = torch.where((p >= 2 * n // 3)[:, None, None] | torch.tensor(not late),
                                  torch.tensor(250, dtype=torch.uint8), vs[at, off])
    query = torch.zeros(2, 4, dk, dtype=dtype)
    query[..., 0] = 1.0
    say(f"attention mxfp4 {dtype} {dk}/{dv} pages of {page}: values of 2^125")
    out, lse = custom_ops.kv_cache_attention(
        query.to(DEV), kc.to(DEV), vc.to(DEV), ks.to(DEV), vs.to(DEV), table.to(DEV),
        torch.tensor(lens, dtype=torch.int32, device=DEV), 1.0, return_lse=True)
    o, z, ob, zb = kv_plain.attention(query, kc, vc, ks, vs, "mxfp4", table, torch.tensor(lens), 1.0)
    kv_plain.near(lse, z, zb, "lse")
    kv_plain.near(out, o, ob, "out")
