"""The small language model with mixers of linear attention: its loss and gradients on the GPU against the host's tensor
operations, serving token by token, tokens drawn from it."""
import copy

import pytest
import torch

import butterfly_amd as tb
from butterfly_amd.sequence_model import ButterflyLM

pytestmark = pytest.mark.gpu


def model(**kw):
    torch.manual_seed(0)
    return ButterflyLM(200, 48, 2, heads=4, **kw)


def test_loss_and_gradients_match_the_host():
    """Against the host in 64 bits.  How far rounding carries is the model's: a head's result is normalised, and where a query and
    a key are nearly at right angles what is normalised is the rounding.  The host's own operations in 32 bits measure it (1e-3
    of the first layer's gradients); the device, whose products and sums are float too, rounds no more than they do: twice
    their distance, and 1e-5 of the largest where theirs happens to be small."""
    host = model()
    gpu, wide = copy.deepcopy(host).cuda(), copy.deepcopy(host).double()
    tokens, target = torch.randint(0, 200, (3, 150)), torch.randint(0, 200, (3, 150))
    target[1, 20:] = -100
    reset = torch.zeros(3, 150, dtype=torch.bool)
    reset[0, 17] = reset[2, 100] = True
    # (same seeds and call numbers: the same dropout masks on all)
    losses = [m.loss(tokens.to(d), target.to(d), reset.to(d)) for m, d in ((host, "cpu"), (gpu, "cuda"), (wide, "cpu"))]
    assert abs(float(losses[1].detach()) - float(losses[2].detach())) < 1e-4 * float(losses[2].detach())
    grads = [torch.autograd.grad(loss, list(m.parameters())) for loss, m in zip(losses, (host, gpu, wide))]
    for (name, _), a, b, c in zip(host.named_parameters(), *grads):
        largest = float(c.abs().max())
        assert float((b.cpu() - c).abs().max()) <= 2 * float((a - c).abs().max()) + 1e-5 * largest, name


def test_token_by_token_gives_the_sequence():
    m = model().cuda().eval()
    tokens = torch.randint(0, 200, (5, 100), device="cuda")
    with torch.no_grad():
        hidden, last = m.hidden(tokens)
        states = m.empty_states(5)
        for t in range(100):
            logits = m.step(tokens[:, t], states)
        want = hidden[:, -1] @ m.embedding.t()
        assert float((logits - want).abs().max()) < 1e-4 * float(want.abs().max())
        for (a, p), (b, q) in zip(states, last):
            assert float((a - b).abs().max()) < 1e-4 * float(b.abs().max())
            assert p.tolist() == q.tolist() == [100] * 5
        # a prompt as one sequence, then on from its states
        _, states = m.hidden(tokens[:, :70])
        rest, _ = m.hidden(tokens[:, 70:99], states)
        _, states = m.hidden(tokens[:, :99])
        assert float((rest - hidden[:, 70:99]).abs().max()) < 1e-4 * float(hidden.abs().max())
        assert float((m.step(tokens[:, 99], states) - want).abs().max()) < 1e-4 * float(want.abs().max())


@pytest.mark.parametrize("heads", [None, 4])
def test_generated_tokens_are_those_of_each_step(heads):
    torch.manual_seed(1)
    m = ButterflyLM(200, 48, 2, heads=heads).cuda().eval()
    prompt, uniform = torch.randint(0, 200, (3, 20), device="cuda"), torch.rand(3, 12, device="cuda")
    temperature = torch.tensor([0.5, 0.0, 1.5], device="cuda")
    tokens = m.generate(prompt, uniform, temperature, top_k=50, top_p=0.9, min_p=0.01)
    assert tokens.shape == (3, 12) and tokens.dtype == torch.int64
    with torch.no_grad():
        states = m.empty_states(3)
        for t in range(20):
            logits = m.step(prompt[:, t], states)
        for t in range(12):
            # every token given those before it; from the second on the logits are the very ones that it was drawn from
            if t > 0:
                logits = m.step(tokens[:, t - 1], states)
            p = torch.softmax(logits[:, :] / temperature.clamp(min=1e-3).unsqueeze(1), 1)
            drawn = tb.sample(logits, uniform[:, t], temperature, 50, 0.9, 0.01)
            # (states by another way: logits off by rounding, a border of the sums may lie between)
            close = (tokens[:, t] == drawn) | (p.gather(1, tokens[:, t:t + 1])[:, 0] > 0)
            assert bool(close.all())
            assert int(tokens[1, t]) == int(logits[1].argmax()) or float(logits[1].max() - logits[1, tokens[1, t]]) < 1e-3


def test_a_training_step_and_a_token_in_graphs():
    m = model(dropout=0.0).cuda()
    tokens, target = (torch.randint(0, 200, (2, 130), device="cuda") for _ in range(2))
    state = m.mixers[0].empty_state(2, "cuda")
    x = torch.randn(2, 48, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.no_grad(), torch.cuda.stream(stream):
        m.mixers[0].step(x, m.mixers[0].empty_state(2, "cuda"))
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph, stream=stream):
        y = m.mixers[0].step(x, state)
    eager = m.mixers[0].empty_state(2, "cuda")
    for s in state:
        s.zero_()
    for _ in range(4):
        x.copy_(torch.randn(2, 48))
        graph.replay()
        with torch.no_grad():
            want = m.mixers[0].step(x, eager)
        torch.cuda.synchronize()
        assert torch.equal(y, want)
        for a, b in zip(state, eager):
            assert torch.equal(a, b)
    # an optimizer's steps: finite gradients for every parameter
    loss = m.loss(tokens, target)
    loss.backward()
    assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in m.parameters())
