"""The loss at the edges of what it is given: what lies behind and between the weight's rows, rows and gradients that are not
finite or of unlike size, empty batches.  Error measure and tolerances are those of the loss's other tests."""
import pytest
import torch

import butterfly_amd as tb
from test_gpu_linear_cross_entropy import DTYPES, check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,features,vocab", [(70, 64, 1000), (300, 72, 1000), (300, 64, 100), (2048, 64, 16390), (3000, 1024, 4100)])
def test_what_lies_behind_the_weight_reaches_nothing(rows, features, vocab, dtype):
    """The last k step of the hidden rows' gradient and the last tile of the logits end inside a step and a tile: NaN behind
    the weight's last row would show in either."""
    hidden, weight, target = make(rows, features, vocab, dtype)
    tall = torch.full((vocab + 300, features), float("nan"), dtype=dtype, device="cuda")
    tall[:vocab] = weight
    for a, b in zip(check(hidden, tall[:vocab], target), check(hidden, weight, target)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
def test_no_rows_give_the_weight_no_gradient(reduction, dtype):
    hidden, weight, target = make(0, 40, 777, dtype)
    # (memory that the operators take next is not zero)
    used = [torch.full((1 << k,), float("nan"), device="cuda") for k in range(8, 22)]
    del used
    h, w = hidden.requires_grad_(), weight.requires_grad_()
    loss = tb.linear_cross_entropy(h, w, target, reduction=reduction)
    dh, dw = torch.autograd.grad(loss, (h, w), torch.ones_like(loss))
    assert dh.shape == (0, 40) and torch.equal(dw, torch.zeros_like(weight))
