"""Launches past HIP's limits are refused on the host: here the gradient's last kernel, which
adds the shares of the sinks' keys (no GPU: nothing is launched)."""
import ctypes

import pytest

from gomlx_hip import _lib

PTR = 1 << 20  # never dereferenced: the call is refused


@pytest.mark.parametrize("B,D,dt", [(1 << 21, 256, _lib.DT_BFLOAT16), (1 << 21, 128, _lib.DT_FLOAT32),
                                    ((1 << 20) + 1, 256, _lib.DT_FLOAT16)])
def test_shares_past_a_launch(B, D, dt):
    s = (ctypes.c_int64 * 3)(256 * D, 256 * D, D)
    with pytest.raises(_lib.BackendError, match="too large") as e:
        _lib.call("ghip_sdpa_window_bwd", dt, *[PTR] * 9, B, 1, 1, 256, 256, D, *[s] * 8, 0, 1, 1, None, 1.0, PTR, 1 << 60,
                  None)
    assert e.value.code == 2
