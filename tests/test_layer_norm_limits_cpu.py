"""Limits of layer norm that need no GPU."""

import ctypes

import pytest

from fast_trimul_b200 import _lib

MOST = (1 << 30) - 1024


@pytest.mark.parametrize("width", [MOST + 1, 1 << 30, 2 ** 31 - 512, 2 ** 31 - 1])
def test_rows_too_wide_for_32_bit_columns_are_refused(width):
    """Columns are counted in 32 bits, those of dw and db together: wider rows ran past 2^31."""
    lib = _lib.load()
    p = ctypes.c_void_p(1 << 20)       # never dereferenced
    assert lib.ftm_layer_norm_fwd(p, 1, width, None, 0, None, 0, 1e-5, p, None, 1, width, None) == _lib.BAD_SHAPE
    assert lib.ftm_layer_norm_bwd(p, 1, width, p, width, p, 0, p, p, p, p, 0, p, 1 << 62, 1, width, None) == _lib.BAD_SHAPE
    assert lib.ftm_layer_norm_bwd_workspace_bytes(1, width) == 0
    assert lib.ftm_layer_norm_bwd_workspace_bytes(1, MOST) == 8 * MOST
