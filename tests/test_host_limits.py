"""Sizes that the operators beside the multiply refuse, and the room they ask for, through the C ABI.  No kernel is launched."""
import ctypes

from butterfly_amd import _capi


def test_masks_of_more_rows_than_the_generator_counts_are_refused():
    """Row 2^32 would drop what row 0 drops."""
    L, one, null = _capi.lib(), ctypes.c_void_p(256), ctypes.c_void_p(0)
    r = _capi.Rowwise(dtype=2, param_dtype=2, rows=(1 << 32) + 1, cols=1, x_stride=1, drop_probability=0.5)
    assert L.bf_rowwise_fw(ctypes.byref(r), one, null, one, null, null, one, null, null, null) == -2
    assert b"2^32" in L.bf_last_error()
    assert L.bf_rowwise_bw_workspace_bytes(ctypes.byref(r)) == _capi.SIZE_INVALID
    # (without dropping the rows need no numbers)
    r.drop_probability = 0.0
    assert L.bf_rowwise_bw_workspace_bytes(ctypes.byref(r)) < _capi.SIZE_INVALID
    r.drop_probability, r.rows = 0.5, 1 << 32
    assert L.bf_rowwise_bw_workspace_bytes(ctypes.byref(r)) < _capi.SIZE_INVALID
