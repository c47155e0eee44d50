"""The small language model converted between types and devices: its positions keep 64 bits."""
import copy

import pytest
import torch

from butterfly_amd.positions import rotary_frequencies
from butterfly_amd.sequence_model import ButterflyLM

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("convert", [lambda m: m.float(), lambda m: m.double().float(), lambda m: m.to(torch.float32), lambda m: m.bfloat16().float(),
                                     lambda m: copy.deepcopy(m.half()).float()])
def test_frequencies_keep_64_bits(convert, device):
    torch.manual_seed(0)
    # (parameters that every conversion leaves as they are)
    m = ButterflyLM(30, 16, 2, heads=2).to(torch.bfloat16).float().eval().to(device)
    tokens, uniform = torch.randint(0, 30, (2, 9), device=device), torch.rand(2, 4).to(device)
    positions = torch.tensor([3, 1 << 24], device=device)
    x = torch.randn(2, 16, device=device)

    def outputs(m):
        with torch.no_grad():
            far = m.mixers[0].step(x, (m.mixers[0].empty_state(2, device)[0], positions.clone()))
            return m.hidden(tokens)[0], m.generate(tokens, uniform, 0.8, top_k=5), far

    want = outputs(m)
    converted = convert(copy.deepcopy(m))
    for mixer in converted.mixers:
        assert mixer.frequencies.dtype == torch.float64 and mixer.frequencies.device.type == device
        assert torch.equal(mixer.frequencies.cpu(), rotary_frequencies(8)[0])
    for a, b in zip(outputs(converted), want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("device", DEVICES)
def test_frequencies_of_ones_own_and_of_no_memory(device):
    m = ButterflyLM(30, 16, 1, heads=2)
    scaled, _ = rotary_frequencies(8, scaling="linear", factor=4.0)
    m.mixers[0].frequencies = scaled
    assert torch.equal(m.to(device).float().mixers[0].frequencies.cpu(), scaled)
    with torch.device("meta"):
        m = ButterflyLM(30, 16, 1, heads=2)
    assert torch.equal(m.to_empty(device=device).mixers[0].frequencies.cpu(), rotary_frequencies(8)[0])
