"""Which kernel a product of 4-bit operands takes (decided on the host, no GPU): every one is reached, and
the sizes that the GPU tests name for one take it."""

import pytest

from mcoplib_amd import _lib

CHOICES = [
    ((1, 512, 5120), "rows"),
    ((1, 8192, 5120), "32x32 by eight waves"),
    ((48, 4099, 5120), "32x32"),
    ((100, 6144, 8192), "64x64 by waves apart"),
    ((64, 16384, 5120), "64x64, three tiles, direct scales"),
    ((2300, 1700, 512), "64x64"),
    ((256, 8192, 5120), "128x64, three tiles, direct scales"),
    ((250, 8100, 5152), "128x64, three tiles"),
    ((1024, 4096, 5120), "128x128, three tiles, direct scales"),
    ((2048, 4096, 4096), "128x128"),
    ((1500, 4096, 4096), "192x128, three tiles, direct scales"),
    ((1237, 4099, 5152), "192x128, three tiles"),
    ((8192, 8192, 8192), "256x256"),
]


@pytest.mark.parametrize("size,form", CHOICES)
def test_every_form_is_chosen_for_some_size(size, form):
    assert _lib.mxfp4_mm_form(*size) == form
    # scales that are not on dwords take registers, nothing else changes
    assert _lib.mxfp4_mm_form(*size, aligned_scales=False) == form.replace(", direct scales", "")


@pytest.mark.parametrize("size", [(0, 64, 64), (64, 0, 64), (64, 64, 0), (64, 64, 48), (-1, 64, 64),
                                  (1, 64, 1 << 31), (1, (1 << 27) + 1, 64), (65535 * 16 + 1, 64, 64)])
def test_no_form_where_nothing_is_launched(size):
    assert _lib.mxfp4_mm_form(*size) == ""


def test_sizes_of_the_gpu_tests():
    from test_gpu_mxfp4_mm_forms import LAST_IN_FIRST_PLACE

    for size in LAST_IN_FIRST_PLACE:
        form = _lib.mxfp4_mm_form(*size)
        last = -(-size[2] // 256) - 1
        assert form.split(",")[0] in ("128x128", "192x128", "256x256"), (size, form)
        assert last % (3 if "three" in form else 2) == 0, (size, form)
    from test_gpu_mxfp4_mm_forms import FORMS

    assert [_lib.mxfp4_mm_form(*size) for size, _ in FORMS] == [form for _, form in FORMS]
    forms = {form for _, form in FORMS}
    assert {form for _, form in CHOICES} <= forms
