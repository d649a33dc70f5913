"""Attention over the quantized cache and the page operators as parts of a program: a decode step through
torch.compile, and what MCOP_DEBUG_TRACE prints of each form that a launch takes."""

import os
import re
import subprocess
import sys

import pytest
import torch

import kv_plain
import mcoplib_amd._C  # noqa: F401
from conftest import ROOT
from gpu_util import DEV, gen, say
from mcoplib import custom_ops

pytestmark = pytest.mark.gpu


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("kind", ["int8", "fp8", "mxfp4"])
def test_a_decode_step_under_torch_compile(kind):
    say(f"decode step {kind} under torch.compile")
    g = gen(5)
    pages, page, heads, group, dim = 20, 16, 2, 4, 64

    class State:
        def __init__(self):
            self.kc, self.ks = (t.to(DEV) for t in kv_plain.empty_cache(kind, pages, page, heads, dim))
            self.vc, self.vs = self.kc.clone(), self.ks.clone()
            self.table = torch.full((6, 4), -1, dtype=torch.int32, device=DEV)
            self.lens = torch.zeros(6, dtype=torch.int32, device=DEV)
            self.counts = torch.zeros(pages, dtype=torch.int32, device=DEV)

        def all(self):
            return (self.kc, self.vc, self.ks, self.vs, self.table, self.lens, self.counts)

    def step(q, k, v, kc, vc, ks, vs, table, lens, counts, who, cu, parents, children):
        ops = torch.ops._C
        slots = torch.empty(k.shape[0], dtype=torch.int64, device=k.device)
        starts, src, dst = torch.empty_like(who), torch.empty_like(parents), torch.empty_like(parents)
        ops.kv_cache_extend(table, lens, counts, who, cu, slots, starts, page)
        ops.kv_cache_write_quant(k, v, kc, vc, ks, vs, slots)
        ops.kv_cache_fork(table, lens, counts, parents, children, src, dst, page)
        ops.kv_cache_copy_pages([kc, vc, ks, vs], src, dst)
        out = torch.empty_like(q)
        lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
        ops.kv_cache_attention(out, q, kc, vc, ks, vs, table, lens, dim ** -0.5, 0, lse)
        ops.kv_cache_free(table, lens, counts, who[:1], page)
        moved = torch.empty(pages // 2, dtype=torch.int32, device=k.device)
        to, used = torch.empty_like(moved), torch.empty_like(moved[:1])
        ops.kv_cache_compact(table, counts, moved, to, used)
        ops.kv_cache_copy_pages([kc, vc, ks, vs], moved, to)
        return out * 2, lse, slots, starts, src, dst, used

    add = [37, 1, 20]
    k, v = (torch.randn(sum(add), heads, dim, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2))
    q = torch.randn(6, heads * group, dim, generator=g).to(torch.bfloat16).to(DEV)
    rest = (_i32([0, 1, 2]), _i32([0, 37, 38, 58]), _i32([0, 2]), _i32([4, 5]))
    eager, compiled = State(), State()
    want = step(q, k, v, *eager.all(), *rest)
    got = torch.compile(step, backend="aot_eager", fullgraph=True)(q, k, v, *compiled.all(), *rest)
    # pages 0 to 2, 3, and 4 and 5; a page more for each fork's end; the first sequence gives one back
    assert want[2].tolist() == [*range(37), 48, *range(64, 84)] and want[6].item() == 7
    for a, b in zip(got + compiled.all(), want + eager.all(), strict=True):
        assert torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))  # NaN too


_SCRIPT = r"""
import sys, torch
sys.path.insert(0, "tests")
from gpu_util import DEV
from mcoplib import custom_ops
ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)
def attend(sequences, heads, queries, dim, page):
    cache = [torch.zeros(64, page, heads, dim, dtype=torch.int8, device=DEV) for _ in range(2)]
    scale = [torch.ones(64, page, heads, device=DEV) for _ in range(2)]
    q = torch.ones(sequences, queries, dim, dtype=torch.bfloat16, device=DEV)
    custom_ops.kv_cache_attention(q, *cache, *scale, ints(*[[0]] * sequences), ints(*[3] * sequences))
    return cache
cache = attend(2, 4, 8, 128, 16)
attend(3, 1, 1, 128, 7)
attend(1, 1, 1, 300, 16)
attend(1, 1, 40000, 64, 16)
custom_ops.kv_cache_copy_pages(cache, ints(0), ints(1))
def pool(rows, columns):
    return (torch.full((rows, columns), -1, dtype=torch.int32, device=DEV), ints(*[0] * rows),
            ints(*[0] * 5000))
few, many = pool(4, 8), pool(2100, 2)
for p, rows in ((few, 4), (many, 2100)):
    who = torch.arange(rows // 2, dtype=torch.int32, device=DEV)
    cu = torch.arange(rows // 2 + 1, dtype=torch.int32, device=DEV)
    custom_ops.kv_cache_extend(*p, who, cu, rows // 2, 16)
    custom_ops.kv_cache_fork(*p, who, who + rows // 2, 16)
custom_ops.kv_cache_free(*few, ints(0), 16)
custom_ops.kv_cache_compact(few[0], few[2])
torch.cuda.synchronize()
print("child ok", flush=True)
"""


def test_every_launch_is_traced():
    say("MCOP_DEBUG_TRACE of attention and the pages")
    env = dict(os.environ, MCOP_DEBUG_TRACE="1")
    out = subprocess.run([sys.executable, "-c", _SCRIPT], cwd=str(ROOT), env=env,
                         capture_output=True, text=True, timeout=100)
    say(out.stdout[-4000:])
    assert out.returncode == 0, out.stderr[-3000:]
    assert "child ok" in out.stdout
    lines = [ln for ln in out.stdout.splitlines() if ln.startswith("[mcop] ")]
    wanted = [r"kv_cache_attention sequences=2 heads=4 of 8 head sizes 128 and 128: matrix, through LDS, kernel",
              r"kv_cache_attention sequences=3 heads=1 of 1 head sizes 128 and 128: matrix kernel, wgs=\d+, 2048 ",
              r"kv_cache_attention sequences=1 heads=1 of 1 head sizes 300 and 300: vector kernel",
              r"kv_cache_attention sequences=1 heads=1 of 40000 .* 1 shares, none split",
              r"kv_cache_copy_pages 2 tensors, 1 pairs, wgs=2",
              r"kv_cache_extend 2 sequences, 2 tokens, 5000 pages, one launch",
              r"kv_cache_fork 2 forks, 5000 pages, one launch",
              r"kv_cache_extend 1050 sequences, 1050 tokens, 5000 pages, two launches",
              r"kv_cache_fork 1050 forks, 5000 pages, two launches",
              r"kv_cache_free 1 sequences",
              r"kv_cache_compact 5000 pages, a table of 4 x 8"]
    for line, want in zip(lines, wanted, strict=True):
        assert re.match(re.escape("[mcop] ") + want, line), (line, want)
