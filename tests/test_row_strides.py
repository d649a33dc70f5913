"""Rows of tensors of three and more dimensions, as the operators with strided inputs take them: dimensions
of size one neither hide rows that are not uniformly strided nor refuse rows that are.  Checks on the CPU
(whose tensors are refused once the strides are accepted), results on the GPU."""

import pytest
import torch

import mx_plain
from gpu_util import DEV, say
from mcoplib_amd import _C

BF = torch.bfloat16
UNIFORM = {
    "last token of a batch": lambda: torch.randn(4, 5, 64)[:, -1:],
    "one of the middle": lambda: torch.randn(3, 2, 5, 64)[:, 1:, 2:3],
    "ones around": lambda: torch.randn(1, 4, 1, 96)[..., :64],
    "two dimensions of a wider row": lambda: torch.randn(4, 5, 96)[..., :64],
    "a row of one": lambda: torch.randn(7, 5, 64)[2:3, 3:4],
    "every other": lambda: torch.randn(2, 6, 64)[:, ::2],
}
OTHER = {
    "a dimension of one before the cut": lambda: torch.randn(2, 1, 5, 64)[:, :, :3],
    "the same, deeper": lambda: torch.randn(2, 1, 1, 5, 64)[:, :, :, 1:4],
    "a cut": lambda: torch.randn(2, 5, 64)[:, :3],
    "swapped": lambda: torch.randn(2, 1, 3, 64).transpose(0, 2),
}


def _calls(x):
    """The operators that take strided rows, on x, and where their codes and scales go."""
    rows = x.numel() // 64
    q, s = torch.zeros(x.shape, dtype=torch.float8_e4m3fn), torch.zeros(rows, 1)
    c, e = (torch.zeros(*x.shape[:-1], n, dtype=torch.uint8) for n in (32, 2))
    move = lambda t: t.to(x.device)  # noqa: E731
    q, s, c, e = map(move, (q, s, c, e))
    r, w = torch.ones(x.shape, dtype=BF, device=x.device), torch.ones(64, dtype=BF, device=x.device)
    return [(lambda: _C.mxfp4_quant(c, x, e), (c, e)),
            (lambda: _C.dynamic_per_token_scaled_fp8_quant(q, x, s), (q, s)),
            (lambda: _C.fused_add_rms_norm(x, r, w, 1e-6), (x, r))]


def _strided(x, device="cpu"):
    """x's values in bf16 at x's own strides."""
    t = torch.empty_strided(x.shape, x.stride(), dtype=BF, device=device)
    return t.copy_(x)


@pytest.mark.parametrize("name", UNIFORM)
def test_uniform_rows_are_taken(name):
    call, _ = _calls(_strided(UNIFORM[name]()))[0]
    with pytest.raises(RuntimeError, match="CUDA"):
        call()


@pytest.mark.parametrize("name", OTHER)
def test_other_rows_are_refused(name):
    call, _ = _calls(_strided(OTHER[name]()))[0]
    with pytest.raises(RuntimeError, match="uniformly strided"):
        call()


@pytest.mark.gpu
@pytest.mark.parametrize("name", OTHER)
def test_other_rows_are_refused_on_the_gpu(name):
    say(f"rows that are not uniformly strided: {name}")
    for call, _ in _calls(_strided(OTHER[name](), DEV)):
        with pytest.raises(RuntimeError, match="uniformly strided"):
            call()


@pytest.mark.gpu
@pytest.mark.parametrize("name", UNIFORM)
def test_uniform_rows_on_the_gpu(name):
    say(f"strided rows: {name}")
    torch.manual_seed(3)
    x = UNIFORM[name]()
    base = _strided(x, DEV)
    plain = base.clone(memory_format=torch.contiguous_format)
    q, e = mx_plain.quant(plain)
    for n, ((call, outs), (same, want)) in enumerate(zip(_calls(base), _calls(plain))):
        call(), same()
        for a, b in zip(outs, want):
            assert mx_plain.same(a.view(torch.uint8) if a.element_size() == 1 else a,
                                 b.view(torch.uint8) if b.element_size() == 1 else b), n
        if n == 0:
            assert torch.equal(outs[0].cpu(), mx_plain.pack(q)) and torch.equal(outs[1].cpu(), e)
    assert not torch.equal(base.cpu(), x.to(BF))  # the last is in place
