"""Linear attention, rotary positions and sampling where offsets pass 2^31 elements and 2^32 bytes: the far end gives what it gives
by itself."""
import pytest
import torch

import butterfly_amd as tb

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def room():
    yield
    torch.cuda.empty_cache()


def test_linear_attention_over_many_steps():
    """4.3e9 values.  A document starts at a chunk's first step, 141 steps from the end: the same products in the same order
    there, but for the segments' cuts (float sums; results rounded once to 8 bits, decays' gradients sums of 24 bits)."""
    steps, heads, d = (1 << 22) + 77, 16, 64
    start = (1 << 22) - 64
    gen = torch.Generator(device="cuda").manual_seed(0)
    q, k = (torch.randn(1, 1, heads, d, generator=gen, device="cuda", dtype=torch.bfloat16).expand(1, steps, heads, d).requires_grad_() for _ in range(2))
    v = torch.randn(1, steps, heads, d, generator=gen, device="cuda", dtype=torch.bfloat16).requires_grad_()
    log_decay = torch.full((1, 1, heads), -0.05, device="cuda").expand(1, steps, heads).requires_grad_()
    reset = torch.zeros(1, steps, dtype=torch.bool, device="cuda")
    reset[0, start] = True
    o, last = tb.linear_attention(q, k, v, log_decay, reset=reset)
    g = torch.randn(1, steps - start, heads, d, generator=gen, device="cuda", dtype=torch.bfloat16)
    full = torch.zeros_like(o)
    full[:, start:] = g
    got = [o.detach()[:, start:], last.detach()] + [x[:, start:] for x in torch.autograd.grad(o, (q, k, v, log_decay), full)]
    del o, full
    parts = [t.detach()[:, start:].clone().requires_grad_() for t in (q, k, v, log_decay)]
    o, last = tb.linear_attention(*parts)
    want = [o.detach(), last.detach(), *torch.autograd.grad(o, parts, g)]
    for name, a, b in zip(("o", "last", "d_q", "d_k", "d_v", "d_log_decay"), got, want):
        a, b = a.double(), b.double()
        if name == "d_log_decay":
            a, b = a[:, 1:], b[:, 1:]   # (a reset step's decay meets nothing; without a state it meets zeros: both are zero)
        assert float((a - b).abs().max()) <= (2.0 ** -8 if name in ("o", "d_q", "d_k", "d_v") else 1e-5) * float(b.abs().max()), name


def test_rotary_of_many_tokens():
    tokens, heads, d = (1 << 20) + 3, 32, 66
    x = torch.zeros(tokens, heads, d, device="cuda", dtype=torch.bfloat16)
    x[-5:] = torch.randn(5, heads, d, device="cuda")
    positions = torch.arange(tokens, device="cuda")
    frequencies, _ = tb.rotary_frequencies(64, device="cuda")
    assert x.numel() > 1 << 31
    for interleaved in (False, True):
        y = tb.rotary(x, positions, frequencies, interleaved)
        assert torch.equal(y[-5:], tb.rotary(x[-5:].clone(), positions[-5:], frequencies, interleaved))
        assert not bool(y[-1000:-5].any())


def test_rows_far_from_each_other():
    room = torch.empty((1 << 31) + 70000, device="cuda", dtype=torch.bfloat16)
    far = room.as_strided((2, 70000), (1 << 31, 1))
    far.copy_(torch.randn(2, 70000, device="cuda"))
    u = torch.tensor([0.3, 0.8], device="cuda")
    assert torch.equal(tb.sample(far, u, top_p=0.9), tb.sample(far.contiguous(), u, top_p=0.9))
    q, k, v = (room.as_strided((2, 70, 2, 64), (1 << 31, 256, 64, 1)) for _ in range(3))
    log_decay = torch.full((2, 70, 2), -0.1, device="cuda")
    o, last = tb.linear_attention(q, k, v, log_decay)
    p, end = tb.linear_attention(q.contiguous(), k.contiguous(), v.contiguous(), log_decay)
    assert torch.equal(o, p) and torch.equal(last, end)
