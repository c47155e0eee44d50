"""Sampling from rows of few possible tokens: every token that the filters leave has to come up, no other.

Weights are off by 2^-37 of themselves on the device and rounded to whole multiples of 2^-44: of a random number and a border between two
tokens, or of a weight and min_p, these tests would have to meet two within some 2^-36 of each other."""
import math

import pytest
import torch

import butterfly_amd as tb

pytestmark = pytest.mark.gpu


def all_kept_come_up(logits, temperature, min_p):
    """One row against evenly spread numbers: the host's tokens, and all of those with w >= min_p among them."""
    # (a kept token's share is min_p / entries at least)
    n = int(math.ceil(2 * int(torch.isfinite(logits).sum()) / min_p))
    u = (torch.arange(n) + 0.5) / n
    got = tb.sample(logits.cuda().expand(n, -1), u.cuda(), temperature=temperature, min_p=min_p).cpu()
    assert torch.equal(got, tb.sample(logits.expand(n, -1), u, temperature=temperature, min_p=min_p))
    x = logits.double()
    kept = torch.exp((x - x.max()) / temperature) >= min_p
    assert sorted(set(got.tolist())) == kept.nonzero()[:, 0].tolist()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("temperature", [1.5, 2.0, 3.0])
def test_the_least_likely_token_passes_min_p(temperature, dtype):
    """Few tokens that a grammar leaves, none of them much less likely than the likeliest: the lowest logit's distance from the
    highest is a rounded number, and what is that far below the highest is not the lowest one."""
    gen = torch.Generator().manual_seed(17)
    for entries in (2, 3, 5, 8):
        for _ in range(12):
            row = torch.full((64,), -math.inf)
            row[torch.randperm(64, generator=gen)[:entries]] = torch.randn(entries, generator=gen) * 2
            all_kept_come_up(row.to(dtype), temperature, 0.02)


@pytest.mark.parametrize("row", [[1.0, -1e-9], [-1e-30, 1.0], [-1.0, 1e-20, 0.0], [0.0, -1e-40], [300.0, 299.0, 1e-6], [-0.96831703, -0.75575686, 0.39087242, 3.0059497, 3.0757267]])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_lowest_logits_beside_zero(row, dtype):
    x = torch.tensor(row, dtype=dtype)
    for min_p in (0.02, 0.3):
        all_kept_come_up(x, 3.0, min_p)
        # (all of them reach a weight, and the lowest is where the search for min_p starts)
        all_kept_come_up(x, 100.0, min_p)
