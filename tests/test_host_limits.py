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


def test_workspace_of_a_loss_of_many_rows():
    """A piece of the vocabulary has 2048 entries at least: 4 KiB a row and 8 of float pairs, whatever the vocabulary."""
    L = _capi.lib()
    for dtype, elem in ((2, 2), (0, 4)):
        for rows in (1 << 16, 1 << 20):
            x = _capi.LinearXent(dtype=dtype, reduction=1, rows=rows, features=1024, vocab=1 << 17, hidden_stride=1024, weight_stride=1024)
            d_l = max(256 << 20, rows * 2048 * elem)
            # d_hidden's sums (one part), d_weight's over the piece (some parts), a number a row
            sums = rows * 1024 * 4 + (64 << 20) + rows * 4
            assert L.bf_linear_xent_bw_workspace_bytes(ctypes.byref(x)) < d_l + sums + (1 << 20)
            x.reduction = 0
            shared = rows * 1024 * 4 if dtype == 0 else 0
            assert L.bf_linear_xent_bw_workspace_bytes(ctypes.byref(x)) < d_l + sums + shared + (1 << 20)
