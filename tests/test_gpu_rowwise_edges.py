"""Norms of rows whose offset is large beside their spread, in the backward pass; generators of several replicas, and ones whose
two numbers are not adjacent; forward calls that a backward pass runs again.  Error measure and tolerances are those of the
row operators' other tests."""
import copy

import pytest
import torch
from torch.utils.checkpoint import checkpoint

import butterfly_amd as tb
from butterfly_amd.sequence_model import ButterflyLM
from test_gpu_rowwise import err, randn, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("offset", [0.0, 1000.0, 10000.0, -30000.0])
@pytest.mark.parametrize("cols", [7, 100, 500, 1000, 2000, 3000, 8000, 9000, 20000])
def test_gradients_of_rows_with_large_offsets(cols, offset):
    """The inputs' own rounding is the reference's too; what is left are roundings of deviations from the row's mean."""
    x = (randn(40, cols, seed=1) + offset).requires_grad_()
    w, b = randn(cols, seed=2, scale=0.3, shift=1.0).requires_grad_(), randn(cols, seed=3).requires_grad_()
    g = randn(40, cols, seed=4)
    y = tb.layer_norm(x, w, b)
    ref = reference(x, g, weight=w, bias=b)
    assert err(y, ref["y"]) < 1e-5
    for got, name in zip(torch.autograd.grad(y, (x, w, b), g, retain_graph=True), ("d_x", "d_weight", "d_bias")):
        assert err(got, ref[name]) < 1e-5, name
    # the parameters' gradients alone
    dw, = torch.autograd.grad(y, w, g)
    assert err(dw, ref["d_weight"]) < 1e-5


@pytest.mark.parametrize("replica", [0, 1, 7, -3, 1 << 40])
def test_replicas_of_a_generator(replica):
    host = torch.tensor([-0x123456789ABCDEF, 0x7FEDCBA987654321])
    device = host.cuda()
    for _ in range(2):
        assert tb.rng_next(device, replica).tolist() == tb.rng_next(host, replica).tolist()
    assert device.tolist() == host.tolist()
    layer = tb.DropoutAdd(0.5, replica=replica).cuda()
    taken = tb.rng_next(layer.rng.clone(), replica)
    x = randn(9, 70, seed=5)
    assert torch.equal(layer(x), tb.dropout_add(x, taken, 0.5))


@pytest.mark.parametrize("reentrant", [False, True])
def test_recomputed_blocks_give_the_gradients_of_kept_ones(reentrant):
    """The same kernels on the same numbers; gradients of the embedding's rows may be added in another order."""
    torch.manual_seed(0)
    kept = ButterflyLM(200, 48, 2, dropout=0.3).cuda()
    again = copy.deepcopy(kept)
    for module in [*again.mixers, *again.mixed, *again.fed]:
        module.forward = (lambda run: lambda *args: checkpoint(run, *args, use_reentrant=reentrant))(module.forward)
    tokens, target = torch.randint(0, 200, (2, 3, 50), device="cuda")
    results = []
    for m in (kept, again):
        for _ in range(2):
            loss = m.loss(tokens, target)
            m.zero_grad()
            loss.backward()
        results.append([loss.detach(), *(p.grad for p in m.parameters()), *m.buffers()])
    for a, b in zip(*results):
        assert float((a.double() - b.double()).abs().max()) <= 1e-6 * float(a.double().abs().max())


def test_a_generator_whose_numbers_are_not_adjacent():
    apart = torch.tensor([[3, 100], [4, 200]], device="cuda")[:, 0]
    x, r, w, b = (randn(*s, seed=k).requires_grad_() for k, s in enumerate(((30, 70), (30, 70), (70,), (70,))))
    results = []
    for rng in (apart, apart.contiguous()):
        y, total = tb.dropout_add_layer_norm(x, rng, 0.5, r, w, b)
        results.append([y, total, *torch.autograd.grad(y, (x, r, w, b), torch.ones_like(y) + total.detach())])
    for a, c in zip(*results):
        assert torch.equal(a, c)
