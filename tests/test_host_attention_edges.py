"""On the host: refusals of the C ABI of linear attention where there are no heads.  No kernel is launched."""
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
