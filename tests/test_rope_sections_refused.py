"""Sections of a rotation that are refused on the host: sums that would wrap around 64 bits."""
import ctypes

import pytest

from gomlx_hip import _lib

PTR = 1 << 20  # never dereferenced: every call here is refused
MOST = 2 ** 63 - 1


@pytest.mark.parametrize("sections", [(MOST, MOST, 34, 0), (MOST, MOST, 2, 32), (2 ** 62, 2 ** 62, 2 ** 62, 2 ** 62), (MOST, 33, 0, 0)])
def test_sections_that_wrap_around(sections):
    axes = 4 if sections[3] else 3 if sections[2] else 2
    r = _lib.Rope(PTR, 0, 8, 1, axes, *sections, PTR, 64, 0)
    s = (ctypes.c_int64 * 3)(2048, 512, 64)
    with pytest.raises(_lib.BackendError, match="the sections hold") as e:
        _lib.call("ghip_rope", _lib.DT_BFLOAT16, PTR, PTR, 1, 4, 8, 64, s, s, r, 0, None)
    assert e.value.code == 1
