"""kv_cache_attention where its numbers end, on the GPU against the formula in 64 bits: weights whose every bit
shows."""

import math

import pytest
import torch

import kv_plain
import mcoplib_amd._C  # noqa: F401
import mx_plain
from gpu_util import DEV, say
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
    and a rounding, 2.25 u of 0.59, so 0.9 u of w, and its own 2 u; two products, in three terms each (to
    2^-26, u / 4), added up in steps of 2 u of the largest, 2: 3 u of 4 at most; w's errors reach half of the 4.
    3 u + (2.9 + 0.25) u / 2 < 5 u; a weight of 17 bits is 2^-19 = 32 u of 4 off.
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
