"""MCOP_DEBUG_TRACE prints the launch decisions of the 4-bit operators and the quantized cache too."""

import os
import re
import subprocess
import sys

import pytest

from conftest import ROOT
from gpu_util import say
from mcoplib_amd import _lib

pytestmark = pytest.mark.gpu

_SCRIPT = r"""
import sys, torch
sys.path.insert(0, "tests")
from gpu_util import DEV
from mcoplib import custom_ops
x = torch.randn(5, 4096, device=DEV).to(torch.bfloat16)
q, s, _ = custom_ops.rms_norm_mxfp4_quant(x, torch.ones_like(x[0]), 1e-6)
wq, ws = custom_ops.mxfp4_quant(torch.randn(512, 4096, device=DEV))
custom_ops.mxfp4_dequant(q, s, torch.float32)
custom_ops.mxfp4_scaled_mm(q, s, wq, ws, torch.bfloat16)
k = torch.randn(5, 4, 128, device=DEV).to(torch.bfloat16)
for heads, at in ((4, slice(None)), (1, slice(0, 1))):
    cache = [torch.zeros(2, 16, heads, 128, dtype=torch.int8, device=DEV) for _ in range(2)]
    scale = [torch.zeros(2, 16, heads, device=DEV) for _ in range(2)]
    custom_ops.kv_cache_write_quant(k[:, at], k[:, at], *cache, *scale, torch.arange(5, device=DEV))
    table = torch.arange(2, dtype=torch.int32, device=DEV)[None]
    cu = torch.tensor([0, 5], dtype=torch.int32, device=DEV)
    custom_ops.kv_cache_read_dequant(*cache, *scale, table, cu, 5, torch.bfloat16)
torch.cuda.synchronize()
print("child ok", flush=True)
"""


def test_every_launch_is_traced():
    say("MCOP_DEBUG_TRACE of the 4-bit operators and the cache")
    env = dict(os.environ, MCOP_DEBUG_TRACE="1")
    out = subprocess.run([sys.executable, "-c", _SCRIPT], cwd=str(ROOT), env=env,
                         capture_output=True, text=True, timeout=100)
    say(out.stdout[-3000:])
    assert out.returncode == 0, out.stderr[-3000:]
    assert "child ok" in out.stdout
    lines = [ln for ln in out.stdout.splitlines() if ln.startswith("[mcop] ")]
    wanted = [r"rms_norm_mxfp4_quant rows=5 hidden=4096 vec=8",
              r"mxfp4_quant rows=512 hidden=4096: .*aligned to 16 bytes, wgs=256",
              r"mxfp4_dequant rows=5 hidden=4096: ",
              r"mxfp4_scaled_mm M=5 N=512 K=4096: " + re.escape(_lib.mxfp4_mm_form(5, 512, 4096)) + "$",
              r"kv_cache_write_quant tokens=5 heads=4 head sizes 128 and 128: whole tokens a wave, 1 ",
              r"kv_cache_read_dequant tokens=5 heads=4 .*whole tokens a wave, 1 ",
              r"kv_cache_write_quant tokens=5 heads=1 .*a vector a group of lanes",
              r"kv_cache_read_dequant tokens=5 heads=1 .*a vector a group of lanes"]
    for line, want in zip(lines, wanted, strict=True):
        assert re.match(re.escape("[mcop] ") + want, line), (line, want)
