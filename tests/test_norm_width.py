"""Widths of layer norm that its kernels' 32-bit column counters do not hold are refused before any launch."""
import ctypes

import pytest

from mace_onegpu import _native as N

BAD = [2 ** 30 + 1, 2 ** 31 - 1024, 2 ** 31 - 1]


@pytest.mark.parametrize("d", BAD)
@pytest.mark.parametrize("dtype", [0, 1, 2])
def test_widths_beyond_the_counters_are_refused(d, dtype):
    L, n = N.lib(), N.c_i64()
    # null pointers: a call that went on would report those instead
    assert L.mace_b200_layer_norm_fwd(None, d, None, None, None, None, None, 1, d, 1e-5, dtype, dtype, None) < 0
    assert b"width %d" % d in L.mace_b200_last_error()
    assert L.mace_b200_layer_norm_bwd(None, d, None, d, None, None, None, None, None, None, None, 1, d, dtype, dtype, None) < 0
    assert b"width %d" % d in L.mace_b200_last_error()
    assert L.mace_b200_layer_norm_bwd_workspace(1, d, ctypes.byref(n)) < 0
    assert b"width %d" % d in L.mace_b200_last_error()
