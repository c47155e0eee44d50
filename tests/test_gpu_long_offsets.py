"""Rows that lie more than 2^31 elements apart in memory, against the same rows close together: the same bits."""
import pytest
import torch

import butterfly_amd as tb

pytestmark = pytest.mark.gpu


def far(rows, stride):
    """The rows of a (n, cols) tensor, `stride` elements apart."""
    n, cols = rows.shape
    wide = torch.empty((n - 1) * stride + cols, dtype=rows.dtype, device="cuda").as_strided((n, cols), (stride, 1))
    assert (n - 1) * stride > 1 << 31
    return wide.copy_(rows)


def same(a, b):
    for x, y in zip(a, b):
        assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows(dtype):
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(33, 130, device="cuda", generator=gen).to(dtype)
    grad = torch.randn(33, 130, device="cuda", generator=gen).to(dtype)
    weight, bias = torch.randn(2, 130, device="cuda", generator=gen).to(dtype)
    rng = torch.tensor([5, 9], device="cuda")

    def run(x, grad):
        x = x.detach().requires_grad_()
        y, total = tb.dropout_add_layer_norm(x, rng, 0.25, x, weight, bias)
        return y, total, *torch.autograd.grad((y, total), x, (grad, grad))

    same(run(far(x, 1 << 27), far(grad, 1 << 27)), run(x, grad))


@pytest.mark.parametrize("dtype,steps", [(torch.float32, 40), (torch.bfloat16, 40), (torch.float32, 1100)])
def test_steps(dtype, steps):
    gen = torch.Generator(device="cuda").manual_seed(2)
    gate, x, grad = torch.randn(3, steps, 70, device="cuda", generator=gen).to(dtype)

    def run(gate, x, grad):
        gate, x = gate[None].detach().requires_grad_(), x[None].detach().requires_grad_()
        h, last = tb.gated_recurrence(gate, x)
        return h, last, *torch.autograd.grad(h, (gate, x), grad[None])

    stride = (1 << 31) // (steps - 1) + 3
    same(run(far(gate, stride), far(x, stride), far(grad, stride)), run(gate, x, grad))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [20, 300])
def test_vocabulary(rows, dtype):
    gen = torch.Generator(device="cuda").manual_seed(3)
    hidden = torch.randn(rows, 64, device="cuda", generator=gen).to(dtype)
    weight = (torch.randn(5000, 64, device="cuda", generator=gen) / 4).to(dtype)
    target = torch.randint(0, 5000, (rows,), device="cuda", generator=gen)

    def run(weight):
        h, w = hidden.detach().requires_grad_(), weight.detach().requires_grad_()
        loss = tb.linear_cross_entropy(h, w, target)
        return loss, *torch.autograd.grad(loss, (h, w))

    same(run(far(weight, 1 << 19)), run(weight))
