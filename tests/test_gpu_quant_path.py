"""The operators as a serving step uses them together: residual add + norm to 4-bit codes, the fused
QKV product, the key heads' norm, the write to the quantized cache and the read of the context; eager,
on another stream, captured and replayed, and through torch.compile."""

import pytest
import torch

import mcoplib_amd._C  # noqa: F401
import mx_plain
from gpu_util import DEV, randn, say, weight
from mcoplib import custom_ops, op

pytestmark = pytest.mark.gpu

H, QH, KH, D, PAGE, EPS = 512, 4, 2, 64, 16, 1e-6
N = (QH + 2 * KH) * D
CODES = {"int8": torch.int8, "fp8": torch.float8_e4m3fn, "mxfp4": torch.uint8}


class Layer:
    def __init__(self, kind, pages=8):
        self.kind = kind
        self.norm = weight(H, 1, torch.bfloat16).to(DEV)
        self.qkv = randn((N, H), 2, torch.bfloat16, scale=0.05)
        self.w = custom_ops.mxfp4_quant(self.qkv.to(DEV))
        self.bias = randn((N,), 3, torch.bfloat16, scale=0.1).to(DEV)
        self.heads = torch.stack([weight(D, 10 + h, torch.bfloat16) for h in range(KH)]).to(DEV)
        width = D // 2 if kind == "mxfp4" else D
        tail = (D // 32,) if kind == "mxfp4" else ()
        sdt = torch.uint8 if kind == "mxfp4" else torch.float32
        self.cache = [torch.zeros(pages, PAGE, KH, width, dtype=CODES[kind], device=DEV)
                      for _ in range(2)]
        self.scale = [torch.zeros(pages, PAGE, KH, *tail, dtype=sdt, device=DEV) for _ in range(2)]

    def step(self, x, residual, slots, table, cu, tokens):
        codes, scale, after = custom_ops.rms_norm_mxfp4_quant(x, self.norm, EPS, residual)
        qkv = custom_ops.mxfp4_scaled_mm(codes, scale, *self.w, torch.bfloat16, self.bias)
        k = qkv[:, QH * D:(QH + KH) * D].unflatten(1, (KH, D)).contiguous()
        v = qkv[:, (QH + KH) * D:].unflatten(1, (KH, D))
        kn = torch.empty_like(k)
        op.head_rms_norm(kn, k, self.heads, EPS, 0, KH)
        custom_ops.kv_cache_write_quant(kn, v, *self.cache, *self.scale, slots)
        return (*custom_ops.kv_cache_read_dequant(*self.cache, *self.scale, table, cu, tokens,
                                                  torch.bfloat16), after, kn, v.contiguous())


def _inputs(T, seed):
    return (randn((T, H), seed, torch.bfloat16).to(DEV),
            randn((T, H), seed + 1, torch.bfloat16).to(DEV))


def _tables(T):
    """Two sequences that share out the T tokens: one page apart, in pages 5, 1, 3, ..."""
    first = T // 3
    table = torch.tensor([[5, 1, 3], [2, 7, 0]], dtype=torch.int32)
    cu = torch.tensor([0, first, T], dtype=torch.int32)
    slots = torch.tensor([int(table[0, p // PAGE]) * PAGE + p % PAGE for p in range(first)]
                         + [int(table[1, p // PAGE]) * PAGE + p % PAGE for p in range(T - first)])
    return slots.to(DEV), table.to(DEV), cu.to(DEV)


@pytest.mark.parametrize("kind", ["int8", "fp8", "mxfp4"])
@pytest.mark.parametrize("T", [1, 45])
def test_one_step(kind, T):
    """The whole step, and each stage against its plain statement on the stage's own input."""
    say(f"quant path {kind} {T} tokens")
    layer = Layer(kind)
    x, r = _inputs(T, 20)
    slots, table, cu = _tables(T)
    key, value, after, kn, v = layer.step(x, r, slots, table, cu, T)
    y, want_after = mx_plain.norm_rows(x, layer.norm, EPS, r)
    assert mx_plain.same(after, want_after)
    a = mx_plain.values(*mx_plain.quant(y))
    b = mx_plain.values(*mx_plain.quant(layer.qkv))
    qkv = a @ b.t() + layer.bias.cpu().double()
    # bf16's rounding (half a step, 2^-8 of the value) and H additions of at most a step of sum|ab| each
    room = 2.0 ** -8 * qkv.abs() + H * 2.0 ** -22 * (a.abs() @ b.abs().t()) + 1e-6
    off = (v.cpu().double().flatten(1) - qkv[:, (QH + KH) * D:]).abs()
    assert bool((off <= room[:, (QH + KH) * D:]).all())
    for got, plain in ((key, kn), (value, v)):
        q, s = mx_plain.vector_codes(plain, kind)
        assert mx_plain.same(got, mx_plain.vector_values(q, s, kind, torch.bfloat16))


@pytest.mark.parametrize("kind", ["int8", "fp8", "mxfp4"])
def test_captured_and_replayed(kind):
    """Captured once, replayed with new inputs and eager work between, each replay equal to the eager
    step on a layer of its own."""
    say(f"quant path graph {kind}")
    T = 33
    layer, eager = Layer(kind), Layer(kind)
    x, r = _inputs(T, 1)
    slots, table, cu = _tables(T)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        layer.step(x, r, slots, table, cu, T)
        with torch.cuda.graph(g, stream=side):
            outs = layer.step(x, r, slots, table, cu, T)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for rep in range(4):
        nx, nr = _inputs(T, 50 + rep)
        x.copy_(nx), r.copy_(nr)
        g.replay()
        want = eager.step(nx, nr, slots, table, cu, T)
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert mx_plain.same(a, b), rep
        assert (nx * 2).sum().item() == (nx * 2).sum().item()


def test_replayed_with_other_tables():
    """Slots, block table and sequence lengths are read when a graph is replayed, not when it is made."""
    T = 33
    layer, eager = Layer("int8"), Layer("int8")
    x, r = _inputs(T, 1)
    slots, table, cu = _tables(T)
    g = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        layer.step(x, r, slots, table, cu, T)
        with torch.cuda.graph(g, stream=side):
            outs = layer.step(x, r, slots, table, cu, T)
    torch.cuda.current_stream().wait_stream(side)
    for first in (0, 5, 32, 33):
        pages = torch.randperm(8, generator=torch.Generator().manual_seed(first)).view(2, 4)
        cpu_slots = [int(pages[0, p // PAGE]) * PAGE + p % PAGE for p in range(first)]
        cpu_slots += [int(pages[1, p // PAGE]) * PAGE + p % PAGE for p in range(T - first)]
        slots.copy_(torch.tensor(cpu_slots))
        table.copy_(pages[:, :3])
        cu.copy_(torch.tensor([0, first, T]))
        g.replay()
        want = eager.step(x, r, slots.clone(), table.clone(), cu.clone(), T)
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert mx_plain.same(a, b), first


def test_on_another_stream():
    """Calls go to the stream that is current, after the work that is queued on it."""
    layer, T = Layer("int8"), 45
    slots, table, cu = _tables(T)
    x, r = _inputs(T, 7)
    want = [t.clone() for t in layer.step(x, r, slots, table, cu, T)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        late = torch.zeros_like(x)
        big = torch.randn(2048, 2048, device=DEV)
        for _ in range(20):
            big = big @ big * 1e-3
        late.copy_(x)
        got = layer.step(late, r, slots, table, cu, T)
    s.synchronize()
    for a, b in zip(got, want):
        assert mx_plain.same(a, b)


def test_torch_compile_aot_eager():
    layer, T = Layer("fp8"), 12
    slots, table, cu = _tables(T)
    x, r = _inputs(T, 3)

    def step(x, r):
        codes = torch.empty(T, H // 2, dtype=torch.uint8, device=DEV)
        scale = torch.empty(T, H // 32, dtype=torch.uint8, device=DEV)
        after = torch.empty_like(x)
        torch.ops._C.rms_norm_mxfp4_quant(codes, x, layer.norm, scale, EPS, r, after)
        out = torch.empty(T, N, dtype=torch.bfloat16, device=DEV)
        torch.ops._C.mxfp4_scaled_mm(out, codes, scale, *layer.w, layer.bias)
        return out, after

    want = step(x, r)
    got = torch.compile(step, backend="aot_eager", fullgraph=True)(x, r)
    for a, b in zip(got, want):
        assert mx_plain.same(a, b)


@pytest.mark.parametrize("kind", ["fp8", "mxfp4"])
def test_torch_compile_of_the_cache(kind):
    """Writes to a cache are seen by the reads behind them, also where the graph is functionalized."""
    layer, other, T = Layer(kind), Layer(kind), 45
    slots, table, cu = _tables(T)
    k = randn((T, KH, D), 5, torch.bfloat16).to(DEV)
    v = randn((T, KH, D), 6, torch.bfloat16).to(DEV)

    def step(k, v, kc, vc, ks, vs):
        torch.ops._C.kv_cache_write_quant(k, v, kc, vc, ks, vs, slots)
        key, value = torch.empty_like(k), torch.empty_like(v)
        torch.ops._C.kv_cache_read_dequant(key, value, kc, vc, ks, vs, table, cu, None)
        return key, value

    want = step(k, v, *layer.cache, *layer.scale)
    got = torch.compile(step, backend="aot_eager", fullgraph=True)(k, v, *other.cache, *other.scale)
    for a, b in zip((*got, *other.cache, *other.scale), (*want, *layer.cache, *layer.scale)):
        assert mx_plain.same(a, b)


def test_two_streams_at_once():
    """The same operators on two streams, on tensors of their own, give what each gives alone."""
    layers = [Layer("int8"), Layer("mxfp4")]
    T = 45
    slots, table, cu = _tables(T)
    x, r = _inputs(T, 9)
    want = [[t.clone() for t in layer.step(x, r, slots, table, cu, T)] for layer in layers]
    streams = [torch.cuda.Stream() for _ in layers]
    got = []
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, layer in zip(streams, layers):
            with torch.cuda.stream(s):
                got.append(layer.step(x, r, slots, table, cu, T))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        for s, t in zip(a, b):
            assert mx_plain.same(s, t)


@pytest.mark.parametrize("kind", ["int8", "fp8", "mxfp4"])
def test_replays_among_other_allocations(kind):
    """Between replays other work allocates tensors of the step's sizes, fills them with bytes that spoil
    whatever reads them, and frees them: each replay still gives the eager step's results, and touches
    none of those tensors."""
    say(f"quant path graph among allocations {kind}")
    T = 33
    layer, eager = Layer(kind), Layer(kind)
    x, r = _inputs(T, 1)
    slots, table, cu = _tables(T)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        layer.step(x, r, slots, table, cu, T)
        with torch.cuda.graph(g, stream=side):
            outs = layer.step(x, r, slots, table, cu, T)
    torch.cuda.current_stream().wait_stream(side)
    sizes = [t.numel() * t.element_size() for t in outs]
    sizes += [T * H // 2, T * H // 32, T * N * 2, T * KH * D * 2]  # what the step makes on its way
    held = []
    for rep in range(4):
        nx, nr = _inputs(T, 50 + rep)
        want = [t.clone() for t in eager.step(nx, nr, slots, table, cu, T)]
        held = [torch.full((n,), 255, dtype=torch.uint8, device=DEV) for n in sizes for _ in range(3)]
        x.copy_(nx), r.copy_(nr)
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert mx_plain.same(a, b), rep
        assert all(bool((t == 255).all()) for t in held), rep
        if rep % 2:
            held = []  # the next round's go where these lay
