"""The small language model's answers where no token can be drawn."""
import math

import pytest
import torch

from butterfly_amd.sequence_model import ButterflyLM


@pytest.mark.parametrize("heads", [None, 2])
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_sequences_without_a_possible_token(heads, device):
    """A sequence whose logits are all NaN has no tokens: -1 from there on, which is never looked up, and the others are as they
    are without it."""
    torch.manual_seed(2)
    m = ButterflyLM(30, 16, 2, heads=heads).eval().to(device)
    with torch.no_grad():
        m.embedding[7] = math.nan
    prompt = torch.tensor([[1, 2, 3, 4], [5, 7, 9, 11], [8, 8, 8, 8]], device=device)
    uniform = torch.rand(3, 6, generator=torch.Generator().manual_seed(0)).to(device)
    tokens = m.generate(prompt, uniform, 0.0)
    assert tokens[1].tolist() == [-1] * 6
    assert bool((tokens[[0, 2]] >= 0).all()) and not bool((tokens == 7).any())
    assert torch.equal(tokens[[0, 2]], m.generate(prompt[[0, 2]], uniform[[0, 2]], 0.0))
    # drawn tokens, settings of each sequence
    drawn = m.generate(prompt, uniform, torch.tensor([0.0, 1.0, 0.0], device=device), top_k=5, top_p=0.9)
    assert torch.equal(drawn[0], tokens[0]) and drawn[1].tolist() == [-1] * 6
