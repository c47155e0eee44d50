"""The small language model's answers, token by token, and its training step in a graph."""
import copy

import pytest
import torch
from torch.nn import functional as F

import butterfly_amd as tb
from butterfly_amd.sequence_model import ButterflyLM

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads", [None, 4])
@pytest.mark.parametrize("settings", [{}, {"temperature": 0.7}, {"top_k": 5}, {"top_p": 0.6}, {"min_p": 0.2}, {"temperature": "rows", "top_k": 50, "top_p": 0.9, "min_p": 0.01}])
def test_generated_tokens_are_drawn_from_the_logits_of_each_step(heads, settings):
    """The very tokens: the prompt's states and logits come as generate() has them, so that all numbers are the same ones."""
    torch.manual_seed(1)
    m = ButterflyLM(200, 48, 2, heads=heads).cuda().eval()
    prompt, uniform = torch.randint(0, 200, (3, 20), device="cuda"), torch.rand(3, 12, device="cuda")
    if settings.get("temperature") == "rows":
        settings = {**settings, "temperature": torch.tensor([0.5, 0.0, 1.5], device="cuda")}
    tokens = m.generate(prompt, uniform, **settings)
    assert tokens.shape == (3, 12) and tokens.dtype == torch.int64
    with torch.no_grad():
        hidden, states = m.hidden(prompt)
        logits = F.linear(hidden[:, -1], m.embedding)
        for t in range(12):
            if t > 0:
                logits = m.step(tokens[:, t - 1], states)
            assert torch.equal(tokens[:, t], tb.sample(logits, uniform[:, t], **settings)), t
    # other numbers give other tokens: they are not the likeliest ones alone
    if settings.get("temperature") is None and "top_k" not in settings:
        assert not torch.equal(tokens, m.generate(prompt, 1 - uniform, **settings))


@pytest.mark.parametrize("heads", [None, 4])
def test_a_training_step_in_a_graph(heads):
    """Loss and every parameter's gradient, replayed with other parameters and tokens, against the eager step."""
    torch.manual_seed(0)
    m = ButterflyLM(200, 48, 2, heads=heads, dropout=0.0).cuda()
    eager = copy.deepcopy(m)
    tokens, target = (torch.randint(0, 200, (2, 130), device="cuda") for _ in range(2))

    def step(model, tokens, target):
        loss = model.loss(tokens, target)
        return [loss.detach(), *torch.autograd.grad(loss, list(model.parameters()))]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for _ in range(2):
            step(m, tokens, target)
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = step(m, tokens, target)
    gen = torch.Generator().manual_seed(5)
    for n in range(4):
        with torch.no_grad():
            for p, q in zip(m.parameters(), eager.parameters()):
                p.mul_(0.9)
                q.copy_(p)
            for t in (tokens, target):
                t.copy_(torch.randint(0, 200, (2, 130), generator=gen))
        for t in out:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        want = step(eager, tokens, target)
        torch.cuda.synchronize()
        for (name, _), a, b in zip([("loss", None), *m.named_parameters()], out, want):
            # float32; the embedding's gradient is summed by a library in an order of its own
            assert float((a - b).abs().max()) <= 1e-5 * float(b.abs().max()), (n, name)
