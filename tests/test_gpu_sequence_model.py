"""The small language model on butterfly layers: its loss and gradients on the GPU against the host's tensor operations,
training, and serving token by token."""
import copy

import pytest
import torch

import butterfly_amd as tb
from butterfly_amd.sequence_model import ButterflyLM

pytestmark = pytest.mark.gpu


def model(**kw):
    torch.manual_seed(0)
    return ButterflyLM(200, 48, 2, **kw)


def test_loss_and_gradients_match_the_host():
    host = model()
    gpu = copy.deepcopy(host).cuda()
    tokens, target = torch.randint(0, 200, (3, 50)), torch.randint(0, 200, (3, 50))
    target[1, 20:] = -100
    reset = torch.zeros(3, 50, dtype=torch.bool)
    reset[0, 17] = True
    # (same seeds and call numbers: the same dropout masks on both)
    losses = [m.loss(tokens.to(d), target.to(d), reset.to(d)) for m, d in ((host, "cpu"), (gpu, "cuda"))]
    # float32 on both sides through some twenty layers
    assert abs(float(losses[0]) - float(losses[1])) < 1e-4 * float(losses[0])
    grads = [torch.autograd.grad(loss, list(m.parameters())) for loss, m in zip(losses, (host, gpu))]
    for a, b in zip(*grads):
        assert float((a - b.cpu()).abs().max()) < 1e-3 * max(float(a.abs().max()), 1e-6)
    for a, b in zip(host.buffers(), gpu.buffers()):
        assert torch.equal(a, b.cpu())


def test_token_by_token_gives_the_sequence():
    m = model().cuda().eval()
    tokens = torch.randint(0, 200, (5, 30), device="cuda")
    with torch.no_grad():
        hidden, last = m.hidden(tokens)
        states = m.empty_states(5)
        for t in range(30):
            logits = m.step(tokens[:, t], states)
        want = hidden[:, -1] @ m.embedding.t()
    assert float((logits - want).abs().max()) < 1e-4 * float(want.abs().max())
    for a, b in zip(states, last):
        assert float((a - b).abs().max()) < 1e-4 * float(b.abs().max())
    # a prompt as one sequence, then on from its states
    with torch.no_grad():
        _, states = m.hidden(tokens[:, :29])
    assert float((m.step(tokens[:, 29], states) - want).abs().max()) < 1e-4 * float(want.abs().max())


def test_training_lowers_the_loss():
    m = model(dropout=0.05).cuda()
    tokens = torch.arange(40, device="cuda").repeat(4, 1)
    optimizer = torch.optim.Adam(m.parameters(), 1e-2)
    losses = []
    for _ in range(30):
        loss = m.loss(tokens[:, :-1], tokens[:, 1:])
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        losses.append(float(loss))
    assert losses[-1] < 0.5 * losses[0]
    assert tb.DropoutAddLayerNorm is type(m.mixed[0]) and int(m.mixed[0].rng[1]) == 30
