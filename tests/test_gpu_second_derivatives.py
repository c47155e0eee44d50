"""Gradients that are to be differentiated again: dropout with its sum has second derivatives, the other operators beside the multiply
say that they have none instead of counting as constants."""
import pytest
import torch

import butterfly_amd as tb
from butterfly_amd.rowwise import dropout_mask

pytestmark = pytest.mark.gpu

RNG = (5, 6)


def randn(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).cuda().requires_grad_()


def operators():
    rng = torch.tensor(RNG, device="cuda")
    x, gate, w, b, r = randn(4, 40, seed=1), randn(2, 3, 8, seed=2), randn(40, seed=3), randn(40, seed=4), randn(4, 40, seed=5)
    v, state = randn(2, 3, 8, seed=6), randn(2, 8, seed=7)
    weight, target = randn(30, 40, seed=8), torch.tensor([1, 2, -100, 29], device="cuda")
    many, targets = randn(80, 40, seed=9), torch.arange(80, device="cuda") % 30
    return {
        "layer_norm": (lambda: tb.layer_norm(x, w, b), (x, w, b)),
        "layer_norm of x alone": (lambda: tb.layer_norm(x), (x,)),
        "dropout_add_layer_norm": (lambda: tb.dropout_add_layer_norm(x, rng, 0.3, r, w, b)[0], (x, r, w, b)),
        "both results": (lambda: torch.cat(tb.dropout_add_layer_norm(x, rng, 0.3, r, w, b)), (x, r, w, b)),
        "gated_recurrence": (lambda: tb.gated_recurrence(gate, v, state)[0], (gate, v, state)),
        "its last state": (lambda: tb.gated_recurrence(gate, v, state)[1], (gate, v, state)),
        "linear_cross_entropy": (lambda: tb.linear_cross_entropy(x, weight, target), (x, weight)),
        "frozen weight": (lambda: tb.linear_cross_entropy(x, weight.detach(), target, reduction="none"), (x,)),
        "many rows": (lambda: tb.linear_cross_entropy(many, weight, targets), (many, weight)),
    }


@pytest.mark.parametrize("name", ["layer_norm", "layer_norm of x alone", "dropout_add_layer_norm", "both results", "gated_recurrence",
                                  "its last state", "linear_cross_entropy", "frozen weight", "many rows"])
def test_no_second_derivative_is_said(name):
    run, leaves = operators()[name]
    out = run()
    once = torch.autograd.grad(out, leaves, torch.ones_like(out))
    # (asking for a graph alone changes nothing)
    out = run()
    grads = torch.autograd.grad(out, leaves, torch.ones_like(out), create_graph=True)
    for a, b in zip(once, grads):
        assert torch.equal(a, b)
    total = sum(g.square().sum() for g in grads)
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(total, leaves, allow_unused=True)
    # through the incoming gradient as well
    up = torch.ones_like(out).requires_grad_()
    grads = torch.autograd.grad(run(), leaves, up, create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(sum(g.sum() for g in grads), up)


def test_dropout_add_has_second_derivatives():
    rng, p = torch.tensor(RNG, device="cuda"), 0.25
    x, r = randn(9, 33, seed=10), randn(9, 33, seed=11)
    factor = dropout_mask(rng, 9, 33, p) * (65536 / 49152)
    y = tb.dropout_add(x, rng, p, r)
    dx, dr = torch.autograd.grad((y ** 3).sum(), (x, r), create_graph=True)
    got = torch.autograd.grad((dx * dr).sum(), (x, r))
    # d = 3 y^2: sum of d factor d, by y: 36 y^3 factor
    want = 36 * y.detach().double() ** 3 * factor
    for a, b in zip(got, (want * factor, want)):
        assert float((a.double() - b).abs().max() / b.abs().max()) < 1e-6
    y, total = tb.dropout_add_layer_norm(x, rng, p, r)
    dx, = torch.autograd.grad((total ** 2).sum(), x, create_graph=True)
    second, = torch.autograd.grad(dx.sum(), x)
    assert float((second.double() - 2 * factor.double() ** 2).abs().max()) < 1e-6
