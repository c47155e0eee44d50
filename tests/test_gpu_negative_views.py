"""Imaginary parts of conjugates: views whose memory holds the opposite of what they are.  A single column needs no copy for its
stride, so nothing else would look at the sign."""
import pytest
import torch

import butterfly_amd as tb

pytestmark = pytest.mark.gpu


def view(*shape, seed=0):
    """(a negative view, the same numbers in memory of their own)"""
    z = torch.randn(*shape, dtype=torch.complex64, generator=torch.Generator().manual_seed(seed)).cuda()
    v = z.conj().imag
    assert v.is_neg()
    return v, (-z.imag).contiguous()


def test_rows():
    (x, x0), (r, r0), (g, g0) = (view(9, 1, seed=k) for k in range(3))
    (w, w0), (b, b0) = (view(1, seed=k) for k in (3, 4))
    rng = torch.tensor([1, 2], device="cuda")
    for args, grad in (((x, r, w, b), g), ((x0, r0, w0, b0), g0)):
        leaves = [t.detach().requires_grad_() for t in args]
        y, total = tb.dropout_add_layer_norm(leaves[0], rng, 0.5, *leaves[1:])
        out = [y, total, tb.dropout_add(leaves[0], rng, 0.5), tb.layer_norm(leaves[0], leaves[2], leaves[3]),
               *torch.autograd.grad((y, total), leaves, (grad, grad))]
        if args[0] is x:
            first = out
    for a, c in zip(first, out):
        assert torch.equal(a, c)


def test_recurrence():
    (z, z0), (x, x0), (g, g0) = (view(2, 30, 1, seed=k) for k in range(3))
    (s, s0), (gl, gl0) = (view(2, 1, seed=k) for k in (3, 4))
    results = []
    for args, grads in (((z, x, s), (g, gl)), ((z0, x0, s0), (g0, gl0))):
        leaves = [t.detach().requires_grad_() for t in args]
        h, last = tb.gated_recurrence(*leaves)
        with torch.no_grad():
            step = tb.gated_recurrence_step(args[0][:, 0], args[1][:, 0], s0.clone())
        results.append([h, last, step, *torch.autograd.grad((h, last), leaves, grads)])
    for a, b in zip(*results):
        assert torch.equal(a, b)
    with pytest.raises(RuntimeError, match="in place"):
        tb.gated_recurrence_step(z0[:, 0], x0[:, 0], s)


@pytest.mark.parametrize("rows", [1, 90])
def test_loss(rows):
    (h, h0), (w, w0) = view(rows, 1), view(300, 1, seed=1)
    target = torch.arange(rows, device="cuda")
    results = []
    for args in ((h, w), (h0, w0)):
        leaves = [t.detach().requires_grad_() for t in args]
        loss = tb.linear_cross_entropy(*leaves, target)
        results.append([loss, *torch.autograd.grad(loss, leaves)])
    for a, b in zip(*results):
        assert torch.equal(a, b)
