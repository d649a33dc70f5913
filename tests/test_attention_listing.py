"""The attention kernels that take codes through LDS by direct loads, read from the assembly that the build's
flags give (no GPU): each direct load has its LDS address, and none is started while the wave's own LDS reads,
which may be of the buffer that it fills, are outstanding on any path."""

import re
import subprocess

import pytest

from conftest import ROOT
from test_build_resources import _build_module
from test_lds_barriers import _kernels, unwaited_barriers

UNITS = ["kv_attention_int8", "kv_attention_fp8", "kv_attention_mxfp4"]


@pytest.fixture(scope="module", params=UNITS)
def built(request, tmp_path_factory):
    b = _build_module()
    try:
        subprocess.run([b.HIPCC, "--version"], capture_output=True, check=True)
    except (OSError, subprocess.CalledProcessError):
        pytest.skip(f"{b.HIPCC} not available")
    out = tmp_path_factory.mktemp("listing") / "unit.s"
    r = subprocess.run([b.HIPCC, *b.COMPILE_FLAGS, "-S", "--cuda-device-only",
                        str(ROOT / "mcoplib_amd" / "csrc" / f"{request.param}.hip"), "-o", str(out)],
                       capture_output=True, text=True, check=True, timeout=300)
    kernels = {n: k for n, k in _kernels(out.read_text()).items() if "k_kv_attention_lines" in n}
    assert len(kernels) == 12  # four shapes, three types
    return kernels, r.stderr


def test_direct_loads_have_their_lds_address(built):
    kernels, said = built
    assert "reserved register" not in said, said[:500]
    for name, lines in kernels.items():
        writes, loads = 0, 0
        for ln in lines:
            if re.match(r"s_\w+ m0,", ln):
                writes += 1
            elif "global_load_lds" in ln:
                assert writes == 1, (name, ln, writes)
                writes, loads = 0, loads + 1
        assert loads > 0, name


def test_no_direct_load_starts_with_lds_reads_in_flight(built):
    kernels, _ = built
    bad = {}
    for name, lines in kernels.items():
        # a direct load in a barrier's place: what may be outstanding there
        found = unwaited_barriers(["s_barrier" if "global_load_lds" in ln else ln for ln in lines])
        if found:
            bad[name] = found
    assert not bad, bad


def test_codes_are_read_as_lds(built):
    """No generic-address access: those would wait for both memories."""
    for name, lines in built[0].items():
        assert not any(ln.startswith("flat_") for ln in lines), name
