"""On the host: rotary positions, linear attention and sampling composed from tensor operations, against their formulas
and differences; the C ABI's refusals and size queries of the same operators.  No kernel is launched."""
import ctypes
import math

import pytest
import torch

import butterfly_amd as tb


def test_rotary():
    frequencies, magnitude = tb.rotary_frequencies(6)
    assert magnitude == 1.0 and torch.allclose(frequencies, torch.tensor([1.0, 10000.0 ** (-1 / 3), 10000.0 ** (-2 / 3)]).double())
    x = torch.randn(2, 5, 3, 8, dtype=torch.float64)
    positions = torch.tensor([[0, 1, 2, 3, 4], [7, 0, 100, 5, 5]])
    for interleaved in (False, True):
        y = tb.rotary(x, positions, frequencies, interleaved, 1.25)
        for b, t, h, p in ((0, 3, 1, 0), (1, 2, 2, 1), (1, 0, 0, 2)):
            i, j = (2 * p, 2 * p + 1) if interleaved else (p, p + 3)
            angle = float(positions[b, t] * frequencies[p])
            a, c = float(x[b, t, h, i]), float(x[b, t, h, j])
            assert abs(float(y[b, t, h, i]) - 1.25 * (a * math.cos(angle) - c * math.sin(angle))) < 1e-12
            assert abs(float(y[b, t, h, j]) - 1.25 * (a * math.sin(angle) + c * math.cos(angle))) < 1e-12
        assert torch.equal(y[..., 6:], x[..., 6:])
        leaf = x.clone().requires_grad_()
        assert torch.autograd.gradcheck(lambda v: tb.rotary(v, positions, frequencies, interleaved, 1.25), leaf)


def test_rotary_frequencies():
    plain, _ = tb.rotary_frequencies(64)
    linear, one = tb.rotary_frequencies(64, scaling="linear", factor=4.0)
    assert one == 1.0 and torch.equal(linear, plain / 4)
    based, _ = tb.rotary_frequencies(64, scaling="base", factor=4.0)
    assert float(based[0]) == 1.0 and abs(float(based[-1] / plain[-1]) - 0.25) < 1e-12
    parts, magnitude = tb.rotary_frequencies(64, scaling="parts", factor=16.0, context=2048)
    turns = plain * 2048 / (2 * math.pi)
    assert torch.equal(parts[turns >= 32], plain[turns >= 32]) and torch.allclose(parts[turns <= 1], plain[turns <= 1] / 16, rtol=1e-15)
    between = (turns > 1) & (turns < 32)
    assert bool((parts[between] < plain[between]).all()) and bool((parts[between] > plain[between] / 16).all())
    assert abs(magnitude - (0.1 * math.log(16) + 1)) < 1e-15
    for kw in (dict(rotated=7), dict(rotated=0), dict(rotated=8, scaling="other"), dict(rotated=8, scaling="linear", factor=0.5),
               dict(rotated=8, scaling="parts", factor=2.0), dict(rotated=8, scaling="parts", factor=2.0, context=10, fast=1.0, slow=1.0)):
        with pytest.raises(ValueError):
            tb.rotary_frequencies(**kw)


def test_linear_attention():
    gen = torch.Generator().manual_seed(0)
    q, k, v, state = (torch.randn(*s, dtype=torch.float64, generator=gen).requires_grad_() for s in ((2, 6, 2, 3), (2, 6, 2, 3), (2, 6, 4, 5), (2, 4, 3, 5)))
    log_decay = (-torch.rand(2, 6, 4, dtype=torch.float64, generator=gen)).requires_grad_()
    reset = torch.zeros(2, 6, dtype=torch.bool)
    reset[1, 4] = True
    o, last = tb.linear_attention(q, k, v, log_decay, state, reset, 0.5)
    for b in range(2):
        for h in range(4):
            s = state[b, h].detach().clone()
            for t in range(6):
                s = (0.0 if reset[b, t] else math.exp(float(log_decay[b, t, h])) * s) + torch.outer(k[b, t, h // 2], v[b, t, h]).detach()
                assert (o[b, t, h] - 0.5 * q[b, t, h // 2] @ s).abs().max() < 1e-12
            assert (last[b, h] - s).abs().max() < 1e-12
    assert torch.autograd.gradcheck(lambda *a: tb.linear_attention(*a, reset, 0.5), (q, k, v, log_decay, state))
    with torch.no_grad():
        whole, last = tb.linear_attention(q, k, v, log_decay, state)
        s = state.clone()
        for t in range(6):
            out = tb.linear_attention_step(q[:, t], k[:, t], v[:, t], log_decay[:, t], s)
            assert torch.allclose(out, whole[:, t])
        assert torch.allclose(s, last)
    with pytest.raises(RuntimeError):
        tb.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], log_decay[:, 0], state.detach())


def test_sample():
    logits = torch.tensor([[0.0, math.log(2.0), -math.inf, math.log(4.0), math.nan, 0.0]])

    def token(u, **kw):
        return int(tb.sample(logits, torch.tensor([u]), **kw))

    # weights 1 2 0 4 0 1
    assert [token(u) for u in (0.0, 0.124, 0.13, 0.37, 0.38, 0.86, 0.88, 0.999)] == [0, 0, 1, 1, 3, 3, 5, 5]
    assert [token(u, top_k=2) for u in (0.0, 0.32, 0.34)] == [1, 1, 3]
    assert [token(u, top_k=3) for u in (0.1, 0.99)] == [0, 3]      # (the first of the two equal ones)
    assert [token(u, top_p=0.74) for u in (0.1, 0.34)] == [1, 3] and token(0.1, top_p=0.0) == 3
    assert [token(u, min_p=0.4) for u in (0.1, 0.34)] == [1, 3]
    assert token(0.9, temperature=0.0) == 3
    assert tb.sample(torch.full((2, 3), -math.inf), torch.zeros(2)).tolist() == [-1, -1]


def test_operators_refuse_host_tensors():
    ops, x = torch.ops.torch_butterfly, torch.zeros(2, 3, 4, 5)
    for call in (lambda: ops.rotary(x, torch.zeros(2, 3, dtype=torch.int64), torch.zeros(1).double(), False, 1.0),
                 lambda: ops.linear_attention(x, x, x, x[..., 0], None, None, 1.0),
                 lambda: ops.linear_attention_step(x[:, 0], x[:, 0], x[:, 0], x[:, 0, :, 0], torch.zeros(2, 4, 5, 5), 1.0),
                 lambda: ops.sample(x[0, 0], torch.zeros(4), None, 1.0, None, 0, None, 1.0, None, 0.0)):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_c_abi_refuses_bad_descriptors():
    from butterfly_amd import _capi
    L, null, one = _capi.lib(), ctypes.c_void_p(0), ctypes.c_void_p(256)   # (never dereferenced: every call is refused on the host)

    def refused(code, call, text):
        assert call() == code
        assert text in L.bf_last_error(), L.bf_last_error()

    def changed(struct, **kw):
        d = type(struct).from_buffer_copy(struct)
        for k, v in kw.items():
            setattr(d, k, v)
        return d

    a = _capi.LinearAttention(dtype=0, batch=1, steps=1000, heads=4, groups=2, features=64, values=64, scale=1.0)
    kept, work = (getattr(L, "bf_linear_attention_" + n)(ctypes.byref(a)) for n in ("kept_bytes", "fw_workspace_bytes"))
    assert kept == 4 * 16 * 64 * 64 * 4 and 0 < work < _capi.SIZE_INVALID
    back = L.bf_linear_attention_bw_workspace_bytes(ctypes.byref(a))
    assert back >= work + 2 * 1000 * 4 * 64 * 4    # (the gradients of each head)

    def fw(d, ws=one, size=work, keep=null, keep_bytes=0, q=one):
        return lambda: L.bf_linear_attention_fw(ctypes.byref(d), q, one, one, one, null, null, one, null, keep, keep_bytes, ws, size, null)

    def bw(d, ws=one, size=back, keep=one, keep_bytes=kept, dq=one):
        return lambda: L.bf_linear_attention_bw(ctypes.byref(d), one, one, one, one, null, keep, keep_bytes, one, null, dq, one, one, one, null, ws, size, null)

    for kw, code, text in ((dict(dtype=1), -1, b"dtype"), (dict(steps=-1), -1, b"sizes"), (dict(heads=3), -1, b"multiple"), (dict(groups=0), -1, b"multiple"),
                           (dict(features=129), -2, b"128"), (dict(values=200), -2, b"128"), (dict(features=0), -1, b"positive"), (dict(batch=1 << 30), -2, b"2^22"),
                           (dict(steps=(1 << 31) + 1), -2, b"2^31"), (dict(v_stride=(ctypes.c_int64 * 3)(0, -1, 0)), -1, b"strides"),
                           (dict(reset_stride=(ctypes.c_int64 * 2)(0, -1)), -1, b"strides")):
        d = changed(a, **kw)
        refused(code, fw(d), text)
        refused(code, bw(d), text)
        refused(code, lambda: L.bf_linear_attention_step(ctypes.byref(d), one, one, one, one, one, one, null), text)
        for n in ("kept_bytes", "fw_workspace_bytes", "bw_workspace_bytes"):
            assert getattr(L, "bf_linear_attention_" + n)(ctypes.byref(d)) == _capi.SIZE_INVALID
    refused(-4, fw(a, size=work - 1), b"workspace")
    refused(-4, fw(a, ws=null), b"workspace")
    refused(-4, fw(a, ws=ctypes.c_void_p(264)), b"aligned")
    refused(-4, fw(a, keep=one, keep_bytes=kept - 1), b"kept")
    refused(-1, fw(a, q=null), b"NULL")
    refused(-4, bw(a, size=back - 1), b"workspace")
    refused(-4, bw(a, keep=null), b"kept")
    refused(-4, bw(a, keep_bytes=kept - 1), b"kept")
    refused(-4, bw(a, keep=ctypes.c_void_p(264)), b"aligned")
    refused(-1, bw(a, dq=null), b"NULL")
    refused(-1, lambda: L.bf_linear_attention_step(ctypes.byref(a), one, one, one, one, null, one, null), b"NULL")
    assert L.bf_linear_attention_fw_workspace_bytes(ctypes.byref(changed(a, batch=64))) == 0
    empty = changed(a, batch=0)
    assert fw(empty, ws=null, size=0)() == 0 and bw(empty, ws=null, size=0, keep=null, keep_bytes=0)() == 0

    r = _capi.Rotary(dtype=0, batch=1, steps=2, heads=3, features=8, rotated=8, magnitude=1.0)
    for kw, code, text in ((dict(dtype=1), -1, b"dtype"), (dict(heads=-1), -1, b"sizes"), (dict(rotated=7), -1, b"even"), (dict(rotated=10), -1, b"at most"),
                           (dict(features=5000, rotated=5000), -2, b"4096"), (dict(x_stride=(ctypes.c_int64 * 3)(-1, 0, 0)), -1, b"strides")):
        d = changed(r, **kw)
        refused(code, lambda: L.bf_rotary_apply(ctypes.byref(d), one, one, one, one, 0, null), text)
    refused(-1, lambda: L.bf_rotary_apply(ctypes.byref(r), null, one, one, one, 0, null), b"NULL")
    refused(-1, lambda: L.bf_rotary_apply(ctypes.byref(r), one, null, one, one, 0, null), b"positions")
    refused(-1, lambda: L.bf_rotary_apply(None, one, one, one, one, 0, null), b"NULL")

    s = _capi.Sample(dtype=0, rows=2, vocab=100, logits_stride=100, temperature=1.0, top_p=1.0)
    for kw, code, text in ((dict(dtype=1), -1, b"dtype"), (dict(rows=-1), -1, b"sizes"), (dict(vocab=0), -1, b"vocab"), (dict(vocab=(1 << 19) + 1), -2, b"2^19"),
                           (dict(rows=1 << 22), -2, b"2^22"), (dict(logits_stride=-1), -1, b"strides")):
        d = changed(s, **kw)
        refused(code, lambda: L.bf_sample_tokens(ctypes.byref(d), one, one, null, null, null, null, one, null), text)
    refused(-1, lambda: L.bf_sample_tokens(ctypes.byref(s), one, null, null, null, null, null, one, null), b"NULL")
    assert L.bf_sample_tokens(ctypes.byref(changed(s, rows=0)), *[null] * 8) == 0


def test_model_with_heads():
    from butterfly_amd.sequence_model import ButterflyLM
    torch.manual_seed(0)
    m = ButterflyLM(50, 16, 2, heads=2, dropout=0.0)
    tokens = torch.randint(0, 50, (2, 9))
    loss = m.loss(tokens[:, :-1], tokens[:, 1:])
    assert all(bool(torch.isfinite(g).all()) for g in torch.autograd.grad(loss, list(m.parameters())))
    m.eval()
    with torch.no_grad():
        hidden, last = m.hidden(tokens)
        states = m.empty_states(2)
        for t in range(9):
            logits = m.step(tokens[:, t], states)
    want = hidden[:, -1] @ m.embedding.t()
    # (float32 through some ten layers)
    assert float((logits - want).detach().abs().max()) < 1e-4 * float(want.detach().abs().max())
    assert m.generate(tokens, torch.rand(2, 4), 0.8, top_k=5).shape == (2, 4)
    with pytest.raises(ValueError, match="multiple"):
        ButterflyLM(50, 18, 1, heads=2)


def test_c_abi_refuses_steps_that_are_too_wide():
    from butterfly_amd import _capi
    L, null, one = _capi.lib(), ctypes.c_void_p(0), ctypes.c_void_p(256)   # (never dereferenced: every call is refused on the host)
    for sizes in (dict(features=128, values=1), dict(features=1, values=128)):
        a = _capi.LinearAttention(dtype=2, batch=1, steps=10, heads=(1 << 15) + 2, groups=2, scale=1.0, **sizes)
        assert L.bf_linear_attention_kept_bytes(ctypes.byref(a)) == _capi.SIZE_INVALID
        assert L.bf_linear_attention_fw(ctypes.byref(a), one, one, one, one, null, null, one, null, null, 0, one, 1 << 40, null) == -2
        assert b"2^22" in L.bf_last_error()
        a.heads = 1 << 15
        # (rows of the states are whole quads of values)
        assert L.bf_linear_attention_kept_bytes(ctypes.byref(a)) == (1 << 15) * sizes["features"] * max(4, sizes["values"]) * 4


def test_sample_settings_at_their_ends():
    logits, u = torch.tensor([[0.0, 1.0, 3.0, 2.0]]), torch.tensor([0.01])
    assert int(tb.sample(logits, u, min_p=math.nan)) == int(tb.sample(logits, u, top_p=math.nan)) == int(tb.sample(logits, u)) == 0
    assert int(tb.sample(logits, u, temperature=math.nan)) == int(tb.sample(logits, u, temperature=1e-300)) == 2
    assert int(tb.sample(logits, torch.tensor([0.3]), temperature=math.inf)) == 1


def test_nothing_to_generate():
    model = tb.sequence_model.ButterflyLM(20, 16, 1, heads=2).eval()
    assert model.generate(torch.tensor([[1, 2, 3]]), torch.zeros(1, 0)).shape == (1, 0)
