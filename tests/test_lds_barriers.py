"""Waits before workgroup barriers, read from the assembly that the build's flags give (no GPU).

A raw s_barrier orders the waves' progress and nothing else: a wave that passes it with LDS reads in
flight lets another wave write over what it still reads, one that passes it with LDS writes in flight
lets another read what is not there yet.  __syncthreads() waits by itself; the product of 4-bit operands
uses the raw barrier, so its kernels are followed here along every path: at each barrier no LDS
instruction may be outstanding."""

import re
import subprocess

import pytest

from conftest import ROOT
from test_build_resources import _build_module

SOURCE = ROOT / "mcoplib_amd" / "csrc" / "mxfp4_mm.hip"


def _kernels(asm):
    """{mangled name: instructions and labels} of the kernels in an assembly listing."""
    out = {}
    for m in re.finditer(r"^(_Z\w+):[^\n]*\n(.*?)^\.Lfunc_end", asm, re.S | re.M):
        lines = [ln.split(";")[0].strip() for ln in m.group(2).splitlines()]
        out[m.group(1)] = [ln for ln in lines
                           if ln and (not ln.startswith(".") or ln.startswith(".LBB"))]
    return out


def _blocks(lines):
    """Basic blocks [(label, instructions)] and their successors by index."""
    blocks = [["", []]]
    for ln in lines:
        if ln.endswith(":"):
            blocks.append([ln[:-1], []])
        else:
            blocks[-1][1].append(ln)
            if re.match(r"s_(c?branch|endpgm|setpc)", ln):
                blocks.append(["", []])
    at = {label: i for i, (label, _) in enumerate(blocks) if label}
    after = []
    for i, (_, ops) in enumerate(blocks):
        last = ops[-1].split() if ops else [""]
        to = [at[last[1]]] if last[0].startswith(("s_branch", "s_cbranch")) else []
        if last[0] not in ("s_branch", "s_endpgm", "s_setpc_b64") and i + 1 < len(blocks):
            to.append(i + 1)
        after.append(to)
    return blocks, after


def unwaited_barriers(lines):
    """The most LDS instructions outstanding at each barrier that some path reaches with any: LDS
    instructions end in order, so lgkmcnt(n) leaves at most n of them."""
    blocks, after = _blocks(lines)
    found = {}

    def through(i, n):
        for k, op in enumerate(blocks[i][1]):
            if op.startswith("ds_"):
                n = min(n + 1, 15)
            elif op.startswith("s_waitcnt") and "lgkmcnt" in op:
                n = min(n, int(re.search(r"lgkmcnt\((\d+)\)", op).group(1)))
            elif op.startswith("s_barrier") and n > 0:
                found[i, k] = max(n, found.get((i, k), 0))
        return n

    entry, todo = {0: 0}, [0]
    while todo:
        i = todo.pop()
        n = through(i, entry[i])
        for j in after[i]:
            if n > entry.get(j, -1):
                entry[j] = n
                todo.append(j)
    return list(found.values())


def test_the_check_finds_reads_that_pass_a_barrier():
    waited = ["ds_read_b128 v[0:3], v9", "s_waitcnt lgkmcnt(0)", "s_barrier", "s_endpgm"]
    assert unwaited_barriers(waited) == []
    assert unwaited_barriers(waited[:1] + waited[2:]) == [1]
    some = ["ds_read_b32 v0, v9", "ds_read_b32 v1, v9 offset:4", "s_waitcnt lgkmcnt(1)", "s_barrier"]
    assert unwaited_barriers(some) == [1]
    # only the path that skips the wait
    paths = ["ds_read_b32 v0, v9", "s_cbranch_scc1 .LBB0_2", "s_waitcnt vmcnt(0) lgkmcnt(0)",
             ".LBB0_2:", "s_barrier", "s_endpgm"]
    assert unwaited_barriers(paths) == [1]
    # a read at the loop's end, waited for at its head only on the way in
    loop = ["s_waitcnt lgkmcnt(0)", ".LBB0_1:", "s_barrier", "ds_read_b32 v0, v9",
            "s_cbranch_scc1 .LBB0_1", "s_endpgm"]
    assert unwaited_barriers(loop) == [15]  # one more each time round, up to what the counter holds


@pytest.fixture(scope="module")
def built(tmp_path_factory):
    """(kernels, what the compiler said) of the product's source under the build's flags."""
    b = _build_module()
    try:
        subprocess.run([b.HIPCC, "--version"], capture_output=True, check=True)
    except (OSError, subprocess.CalledProcessError):
        pytest.skip(f"{b.HIPCC} not available")
    out = tmp_path_factory.mktemp("listing") / "mm.s"
    r = subprocess.run([b.HIPCC, *b.COMPILE_FLAGS, "-S", "--cuda-device-only", str(SOURCE), "-o",
                        str(out)], capture_output=True, text=True, check=True, timeout=300)
    return _kernels(out.read_text()), r.stderr


def test_no_barrier_of_the_product_is_passed_with_lds_in_flight(built):
    kernels, _ = built
    tiles = [n for n in kernels if "k_mxfp4_mm_tile" in n]
    assert len(tiles) >= 27 and all(any("s_barrier" in ln for ln in kernels[n]) for n in tiles)
    bad = {n: u for n, lines in kernels.items() if (u := unwaited_barriers(lines))}
    assert not bad, bad


def test_direct_loads_have_their_lds_address(built):
    """m0 is written once before each direct load, by the compiler, which warns of nothing: a reserved
    register among what inline assembly overwrites is undefined."""
    kernels, said = built
    assert "reserved register" not in said, said[:500]
    for name, lines in kernels.items():
        writes = 0
        for ln in lines:
            if re.match(r"s_\w+ m0,", ln):
                writes += 1
            elif "global_load_lds" in ln:
                assert writes == 1, (name, ln, writes)
                writes = 0
