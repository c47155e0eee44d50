"""More sequences than one dimension of a grid has workgroups for.  Linear gates above one: their products over a run of steps pass the range of the numbers long before a sequence does that has
nothing to be multiplied.  Tolerances are those of the recurrence's other tests."""
import pytest
import torch

import butterfly_amd as tb
from test_gpu_recurrence import TOL, close, make, reference

pytestmark = pytest.mark.gpu

LINEAR = [torch.float32, torch.bfloat16, torch.complex64]


def growing(batch, steps, channels, dtype, first, last, gate):
    """Gates of `gate` in the first and the last steps, where inputs and gradients are zero; none handed in either."""
    v = make(batch, steps, channels, dtype, False)
    v["gate"][:, :first] = v["gate"][:, steps - last:] = gate
    for name in ("x", "grad"):
        v[name][:, :first] = 0
        v[name][:, steps - last:] = 0
    v["state"][:] = 0
    v["grad_last"][:] = 0
    return v


@pytest.mark.parametrize("dtype", LINEAR)
@pytest.mark.parametrize("batch,steps,channels,first,gate", [
    (1, 65537, 64, 3000, 1.25),      # runs of some 64 steps, chunks of 16 of them
    (1, 9000, 70, 2500, 4.0),
    (2, 1111, 66, 300, 1e4),
    (200, 300, 65, 100, 1e6),        # sequences that stay whole: runs of 8 and 4 steps
])
def test_zeros_in_front_stay_zeros_behind_growing_gates(batch, steps, channels, first, gate, dtype):
    v = growing(batch, steps, channels, dtype, first, 0, gate)
    ref = reference(v, False)
    d = {k: t.cuda() for k, t in v.items()}
    for state in (None, d["state"]):
        h, last = tb.gated_recurrence(d["gate"], d["x"], state, None, False)
        assert (h[:, :first] == 0).all()
        close(h, ref["h"], TOL[dtype], "h")
        close(last, ref["last"], 1e-5, "last")


@pytest.mark.parametrize("dtype", LINEAR)
@pytest.mark.parametrize("batch,steps,channels,last,gate", [
    (1, 65537, 64, 3000, 1.25), (1, 9000, 70, 2500, 4.0), (2, 1111, 66, 300, 1e4), (200, 300, 65, 100, 1e6)])
def test_zero_gradients_behind_stay_zero_in_front_of_growing_gates(batch, steps, channels, last, gate, dtype):
    v = growing(batch, steps, channels, dtype, 0, last, gate)
    # (h grows behind: the gates' gradients of those steps are zero times it)
    v["x"][:] = 0
    ref = reference(v, False)
    d = {k: t.cuda() for k, t in v.items()}
    x = d["x"].requires_grad_()
    state = d["state"].requires_grad_()
    h, _ = tb.gated_recurrence(d["gate"], x, state, None, False)
    dx, ds = torch.autograd.grad(h, (x, state), d["grad"])
    assert (dx[:, steps - last:] == 0).all()
    close(dx, ref["d_x"], TOL[dtype], "d_x")
    close(ds, ref["d_state"], 1e-5, "d_state")


@pytest.mark.parametrize("dtype", LINEAR)
def test_a_gate_of_zero_ends_what_grew(dtype):
    """A product of gates that has passed the range meets a zero gate in a later run: the state in front is forgotten."""
    v = growing(1, 9000, 70, dtype, 4000, 0, 4.0)
    v["gate"][:, 3990] = 0
    d = {k: t.cuda() for k, t in v.items()}
    h, last = tb.gated_recurrence(d["gate"], d["x"], None, None, False)
    ref = reference(v, False)
    close(h, ref["h"], TOL[dtype], "h")
    close(last, ref["last"], 1e-5, "last")


def test_more_sequences_than_a_dimension_of_a_grid():
    """Workgroups of 1024 threads: 2^22 of them are 2^32 threads."""
    batch, steps = (1 << 22) + 5, 130
    gen = torch.Generator(device="cuda").manual_seed(1)
    gate, x, grad = (torch.randn(batch, steps, 1, device="cuda", generator=gen) for _ in range(3))
    some = torch.cat((torch.arange(70), torch.arange((1 << 21) - 70, (1 << 21) + 70), torch.arange(batch - 70, batch))).cuda()

    def run(gate, x, grad):
        gate, x = gate.requires_grad_(), x.requires_grad_()
        h, last = tb.gated_recurrence(gate, x)
        return h.detach(), last.detach(), *torch.autograd.grad(h, (gate, x), grad)

    alone = run(gate[some], x[some], grad[some])
    for a, b in zip(run(gate, x, grad), alone):
        assert torch.equal(a[some], b)
