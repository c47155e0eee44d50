"""On the host: refusals of the C ABI of linear attention where there are no heads, of rotary positions where sizes overflow.  No kernel
is launched."""
import ctypes


def test_c_abi_of_groups_without_heads():
    from butterfly_amd import _capi
    L, null, one = _capi.lib(), ctypes.c_void_p(0), ctypes.c_void_p(256)   # (never dereferenced: every call ends on the host)

    def back(d_q, **sizes):
        a = _capi.LinearAttention(**{**dict(dtype=0, batch=1, steps=5, heads=0, groups=2, features=8, values=8, scale=1.0), **sizes})
        return L.bf_linear_attention_bw(ctypes.byref(a), null, null, null, null, null, null, 0, null, null, d_q, one, null, null, null, null, 0, null)

    # the gradients of queries and keys are zeros that have to go somewhere
    assert back(null) == -1 and b"d_q or d_k is NULL" in L.bf_last_error()
    assert back(null, groups=0) == back(null, steps=0) == back(null, batch=0) == 0
    assert back(one, groups=(1 << 22) + 1) == -2 and b"2^22" in L.bf_last_error()


def test_c_abi_refuses_rotary_calls_whose_sizes_overflow():
    from butterfly_amd import _capi
    L, null, one = _capi.lib(), ctypes.c_void_p(0), ctypes.c_void_p(256)   # (never dereferenced: every call is refused on the host)
    for sizes in (dict(batch=1 << 32, steps=1 << 32), dict(batch=1 << 40, steps=1 << 40), dict(batch=1 << 31, steps=(1 << 33) + 1), dict(batch=1 << 30, heads=1 << 20)):
        r = _capi.Rotary(**{**dict(dtype=0, batch=1, steps=2, heads=3, features=8, rotated=8, magnitude=1.0), **sizes})
        assert L.bf_rotary_apply(ctypes.byref(r), one, one, one, one, 0, null) == -2, sizes
        assert b"too many" in L.bf_last_error()
