"""The loss on host tensors does what it does on the device: products of bfloat16 in float, NaN for targets that are no entry of the
vocabulary, a single row without a leading dimension."""
import pytest
import torch

import butterfly_amd as tb


def make(rows, features, vocab, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, features, generator=gen), torch.randn(vocab, features, generator=gen),
            torch.randint(0, vocab, (rows,), generator=gen))


@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
def test_bfloat16_logits_stay_in_float(reduction):
    hidden, weight, target = make(20, 64, 50)
    h, w = hidden.bfloat16(), weight.bfloat16()
    loss = tb.linear_cross_entropy(h, w, target, reduction=reduction)
    assert loss.dtype == torch.float32
    want = torch.nn.functional.cross_entropy(h.double() @ w.double().t(), target, reduction=reduction)
    # logits of some 8 sqrt(features), by sums in float; rounded to bfloat16 they would be off by 2^-9 of themselves
    assert (loss.double() - want).abs().max() < 1e-5 * (1 + want.abs().max())


@pytest.mark.parametrize("ignore", [-100, 0, 7])
@pytest.mark.parametrize("bad", [50, -1, 1 << 40])
def test_targets_outside_the_vocabulary_make_nan(bad, ignore):
    hidden, weight, target = make(20, 16, 50)
    target = target.clamp(min=8)
    target[5], target[6] = bad, ignore
    h, w = hidden.requires_grad_(), weight.requires_grad_()
    each = tb.linear_cross_entropy(h, w, target, ignore, "none")
    assert torch.isnan(each[5]) and each[6] == 0 and torch.isfinite(each[:5]).all() and torch.isfinite(each[7:]).all()
    dh, dw = torch.autograd.grad(each.sum(), (h, w))
    assert torch.isnan(dh[5]).all() and torch.isfinite(dh[:5]).all() and (dh[6] == 0).all() and torch.isnan(dw).all()
    for reduction in ("mean", "sum"):
        assert torch.isnan(tb.linear_cross_entropy(h, w, target, ignore, reduction))


def test_one_row():
    hidden, weight, target = make(3, 16, 50)
    each = tb.linear_cross_entropy(hidden, weight, target, reduction="none")
    one = tb.linear_cross_entropy(hidden[1], weight, target[1], reduction="none")
    assert one.shape == () and torch.allclose(one, each[1])
    assert torch.allclose(tb.linear_cross_entropy(hidden[1], weight, target[1]), each[1])
