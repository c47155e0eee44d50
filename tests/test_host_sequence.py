"""On the host: the operators beside the multiply composed from tensor operations, against the formulas in 64 bits and
differences; the C ABI's refusals and size queries of the same operators.  No kernel is launched."""
import ctypes

import numpy as np
import pytest
import torch

import butterfly_amd as tb
from butterfly_amd.rowwise import dropout_mask


def philox(counter, key):
    """Philox4x32-10 from its definition, with Python's integers."""
    mask = 0xFFFFFFFF
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(b >> 32) ^ c[1] ^ k[0], b & mask, (a >> 32) ^ c[3] ^ k[1], a & mask]
        k = [(k[0] + 0x9E3779B9) & mask, (k[1] + 0xBB67AE85) & mask]
    return c


def test_philox_known_answers():
    # the published test vectors of the generator
    assert philox((0, 0, 0, 0), (0, 0)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = 0xFFFFFFFF
    assert philox((ones,) * 4, (ones,) * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


def test_mask_is_the_generators():
    seed, call, rows, cols = -0x0123456789ABCDEF, 0x7EDCBA9876543210, 5, 21
    rng = torch.tensor([seed, call])
    keep = dropout_mask(rng, rows, cols, 0.3)
    key = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
    for r in range(rows):
        for c in range(cols):
            word = philox((c // 8, r, call & 0xFFFFFFFF, call >> 32), key)[c % 8 // 2]
            bits = word >> 16 if c % 2 else word & 0xFFFF
            assert bool(keep[r, c]) == (bits >= round(65536 * 0.3))


def test_dropout_add_and_norm():
    rng = torch.tensor([3, 4])
    x, r = torch.randn(6, 30, dtype=torch.float64), torch.randn(6, 30, dtype=torch.float64)
    keep = dropout_mask(rng, 6, 30, 0.25)
    want = r + torch.where(keep, x * (65536 / 49152), torch.zeros(()).double())
    assert torch.equal(tb.dropout_add(x, rng, 0.25, r), want)
    assert torch.equal(tb.dropout_add(x, rng, 1.0, r), r)
    w, b = torch.randn(30, dtype=torch.float64), torch.randn(30, dtype=torch.float64)
    y, total = tb.dropout_add_layer_norm(x, rng, 0.25, r, w, b)
    assert torch.equal(total, want)
    assert (y - torch.nn.functional.layer_norm(want, (30,), w, b)).abs().max() < 1e-12
    args = [t.requires_grad_() for t in (x, r, w, b)]
    assert torch.autograd.gradcheck(lambda *a: tb.dropout_add_layer_norm(a[0], rng, 0.25, *a[1:]), args)
    with pytest.raises(ValueError):
        tb.dropout_add(x, rng, 1.5)


@pytest.mark.parametrize("sigmoid", [True, False])
def test_recurrence(sigmoid):
    gate, x, state = (torch.randn(*s, dtype=torch.float64).requires_grad_() for s in ((2, 6, 3), (2, 6, 3), (2, 3)))
    reset = torch.zeros(2, 6, dtype=torch.bool)
    reset[1, 4] = True
    h, last = tb.gated_recurrence(gate, x, state, reset, sigmoid)
    for n in range(2):
        for c in range(3):
            v = float(state[n, c])
            for t in range(6):
                a = float(torch.sigmoid(gate[n, t, c]) if sigmoid else gate[n, t, c])
                v = (0.0 if reset[n, t] else a * v) + (1 - a if sigmoid else 1.0) * float(x[n, t, c])
                assert abs(v - float(h[n, t, c])) < 1e-12
            assert abs(v - float(last[n, c])) < 1e-12
    assert torch.autograd.gradcheck(lambda *a: tb.gated_recurrence(*a, reset, sigmoid), (gate, x, state))
    with torch.no_grad():
        s = state.clone()
        for t in range(4):
            out = tb.gated_recurrence_step(gate[:, t], x[:, t], s, sigmoid)
        want, last = tb.gated_recurrence(gate[:, :4], x[:, :4], state, None, sigmoid)
        assert torch.allclose(out, want[:, 3]) and torch.allclose(s, last)
    with pytest.raises(RuntimeError):
        tb.gated_recurrence_step(gate[:, 0], x[:, 0], state.detach())
    c = torch.randn(1, 4, 2, dtype=torch.complex128).requires_grad_()
    assert torch.autograd.gradcheck(lambda g, v: tb.gated_recurrence(g, v, sigmoid=False), (c, c.detach().clone().requires_grad_()))


def test_loss():
    hidden, weight = torch.randn(2, 7, 5, dtype=torch.float64).requires_grad_(), torch.randn(11, 5, dtype=torch.float64).requires_grad_()
    target = torch.randint(0, 11, (2, 7))
    target[0, 3] = -100
    each = tb.linear_cross_entropy(hidden, weight, target, reduction="none")
    for i, j in np.ndindex(2, 7):
        logits = (weight @ hidden[i, j]).detach()
        want = 0.0 if target[i, j] == -100 else float(torch.log(torch.exp(logits).sum()) - logits[target[i, j]])
        assert abs(float(each[i, j]) - want) < 1e-12
    assert abs(float(tb.linear_cross_entropy(hidden, weight, target)) - float(each.sum()) / 13) < 1e-12
    assert torch.autograd.gradcheck(lambda h, w: tb.linear_cross_entropy(h, w, target, reduction="sum"), (hidden, weight))
    with pytest.raises(ValueError):
        tb.linear_cross_entropy(hidden, weight, target, reduction="max")
    with pytest.raises(ValueError):
        tb.LinearCrossEntropy(5, 11, reduction="max")


def test_operators_refuse_host_tensors():
    ops = torch.ops.torch_butterfly
    x = torch.zeros(2, 3, 4)
    for call in (lambda: ops.layer_norm(x, None, None, 1e-5), lambda: ops.dropout_add(x, None, 0.0, None),
                 lambda: ops.gated_recurrence(x, x, None, None, True), lambda: ops.rng_next(torch.zeros(2, dtype=torch.int64)),
                 lambda: ops.linear_cross_entropy(x, x[0], torch.zeros(2, 3, dtype=torch.int64), -100, 1)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_c_abi_refuses_bad_descriptors():
    from butterfly_amd import _capi
    L, null, one = _capi.lib(), ctypes.c_void_p(0), ctypes.c_void_p(256)   # (never dereferenced: every call is refused on the host)

    def refused(code, call, text):
        assert call() == code
        assert text in L.bf_last_error(), L.bf_last_error()

    r = _capi.Rowwise(dtype=0, param_dtype=0, rows=4, cols=8, x_stride=8)

    def rows(**kw):
        d = _capi.Rowwise.from_buffer_copy(r)
        for k, v in kw.items():
            setattr(d, k, v)
        return lambda: L.bf_rowwise_fw(ctypes.byref(d), one, null, null, null, null, one, null, null, null)

    refused(-1, rows(dtype=1), b"dtype")
    refused(-1, rows(param_dtype=2), b"param_dtype")
    refused(-1, rows(rows=-1), b"sizes")
    refused(-1, rows(x_stride=-1), b"strides")
    refused(-1, rows(drop_probability=1.5), b"drop_probability")
    refused(-1, rows(drop_probability=float("nan")), b"drop_probability")
    refused(-1, rows(drop_probability=0.5), b"rng")
    refused(-1, rows(eps=-1.0), b"eps")
    refused(-2, rows(cols=1 << 30), b"columns")
    refused(-1, lambda: L.bf_rowwise_fw(None, *[null] * 9), b"NULL")
    refused(-1, lambda: L.bf_rowwise_fw(ctypes.byref(r), one, null, null, null, null, null, null, null, null), b"neither")
    refused(-1, lambda: L.bf_rowwise_fw(ctypes.byref(r), one, null, null, one, null, one, null, null, null), b"norm")
    refused(-4, lambda: L.bf_rowwise_bw(ctypes.byref(r), one, one, null, null, null, one, null, null, one, null, null, 0, null), b"workspace")
    assert L.bf_rowwise_bw_workspace_bytes(None) == _capi.SIZE_INVALID
    r.rows = 0
    assert L.bf_rowwise_bw_workspace_bytes(ctypes.byref(r)) == 0
    assert L.bf_rowwise_fw(ctypes.byref(r), *[null] * 9) == 0
    refused(-1, lambda: L.bf_rng_next(null, null, null), b"NULL")

    c = _capi.Recurrence(dtype=0, sigmoid=1, batch=1, steps=4000, channels=64)
    assert 0 < L.bf_recurrence_workspace_bytes(ctypes.byref(c)) < _capi.SIZE_INVALID
    refused(-4, lambda: L.bf_recurrence_fw(ctypes.byref(c), one, one, null, null, one, null, null, 0, null), b"workspace")
    refused(-1, lambda: L.bf_recurrence_fw(ctypes.byref(c), null, one, null, null, one, null, one, 1 << 30, null), b"NULL")
    c.dtype = 1
    refused(-1, lambda: L.bf_recurrence_fw(ctypes.byref(c), one, one, null, null, one, null, one, 1 << 30, null), b"sigmoid")
    c.dtype = 5
    assert L.bf_recurrence_workspace_bytes(ctypes.byref(c)) == _capi.SIZE_INVALID
    c.dtype, c.steps, c.batch = 0, 100, 1000
    assert L.bf_recurrence_workspace_bytes(ctypes.byref(c)) == 0
    c.batch = -1
    refused(-1, lambda: L.bf_recurrence_step(ctypes.byref(c), one, one, one, one, null), b"sizes")

    x = _capi.LinearXent(dtype=0, reduction=1, rows=8, features=16, vocab=100, hidden_stride=16, weight_stride=16, ignore_index=-100)
    need, kept = L.bf_linear_xent_fw_workspace_bytes(ctypes.byref(x)), L.bf_linear_xent_kept_bytes(ctypes.byref(x))
    assert 0 < need < _capi.SIZE_INVALID and 0 < kept < _capi.SIZE_INVALID

    def call(ws, size, weight=one, keep=one, keep_bytes=1 << 40):
        return lambda: L.bf_linear_xent_fw(ctypes.byref(x), one, weight, one, one, keep, keep_bytes, ws, size, null)

    refused(-4, call(one, need - 1), b"workspace")
    refused(-4, call(ctypes.c_void_p(264), need), b"aligned")
    refused(-4, call(one, need, keep_bytes=kept - 1), b"kept")
    refused(-4, call(one, need, keep=null), b"kept")
    refused(-4, call(one, need, keep=ctypes.c_void_p(264)), b"aligned")
    refused(-4, lambda: L.bf_linear_xent_bw(ctypes.byref(x), one, one, one, kept, one, one, null, 0, null), b"workspace")
    refused(-1, call(one, need, weight=ctypes.c_void_p(264)), b"aligned")
    refused(-1, call(one, need, weight=null), b"NULL")
    for field, value, code, text in (("dtype", 1, -1, b"dtype"), ("reduction", 3, -1, b"reduction"), ("vocab", 0, -1, b"vocab"),
                                     ("hidden_stride", -1, -1, b"strides"), ("features", 1 << 20, -2, b"2^16")):
        keep = getattr(x, field)
        setattr(x, field, value)
        refused(code, call(one, 1 << 40), text)
        assert L.bf_linear_xent_bw_workspace_bytes(ctypes.byref(x)) == _capi.SIZE_INVALID
        setattr(x, field, keep)


def test_workspace_of_a_loss_stays_bounded():
    from butterfly_amd import _capi
    L = _capi.lib()
    x = _capi.LinearXent(dtype=2, reduction=1, rows=16384, features=1024, vocab=1 << 20, hidden_stride=1024, weight_stride=1024)
    # the logits' gradient over a piece (256 MiB), d_hidden's sums, two parts of d_weight's piece; the logits would be 32 GiB
    assert L.bf_linear_xent_bw_workspace_bytes(ctypes.byref(x)) < (256 << 20) + (64 << 20) + (64 << 20) + (1 << 20)
    # 16 bytes for each row and 256 entries
    assert L.bf_linear_xent_fw_workspace_bytes(ctypes.byref(x)) < (1 << 30) + (1 << 20)
    # hidden; weights that 16 bytes do not divide have room for a copy too
    assert L.bf_linear_xent_kept_bytes(ctypes.byref(x)) < (32 << 20) + (1 << 20)
    x.features = x.weight_stride = 1023
    assert L.bf_linear_xent_kept_bytes(ctypes.byref(x)) > (2 << 30)
