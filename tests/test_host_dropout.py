"""Dropout modules in several processes, as copies in forward calls that a backward pass runs again, and in bfloat16, on the
host."""
import copy
import os
import tempfile

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp
from torch.utils.checkpoint import checkpoint

import butterfly_amd as tb
from butterfly_amd.rowwise import dropout_mask


def _rank(rank, path):
    dist.init_process_group("gloo", init_method=f"file://{path}/store", rank=rank, world_size=2)
    try:
        torch.manual_seed(rank)
        model = torch.nn.Sequential(torch.nn.Linear(32, 32), tb.DropoutAdd(0.5), tb.DropoutAdd(0.5, replica=0))
        model = torch.nn.parallel.DistributedDataParallel(model)
        for _ in range(2):
            model(torch.ones(16, 32)).sum().backward()
        layers = list(model.module)[1:]
        rng, state = layers[0].rng.clone(), layers[0].state_dict()
        state = {k: v.clone() for k, v in state.items()}
        torch.save(([layer(torch.ones(16, 32)) for layer in layers], rng, state), f"{path}/{rank}")
    finally:
        dist.destroy_process_group()


def test_ranks_drop_elements_of_their_own():
    """DistributedDataParallel gives every rank the first one's seeds."""
    with tempfile.TemporaryDirectory() as path:
        os.environ.setdefault("OMP_NUM_THREADS", "2")
        mp.spawn(_rank, (path,), nprocs=2)
        (first, rng, state), (second, other_rng, _) = (torch.load(f"{path}/{rank}", weights_only=True) for rank in range(2))
    assert torch.equal(rng, other_rng) and int(rng[1]) == 2
    # a share of 512 independent draws: five standard deviations
    assert abs(float((first[0] == second[0]).float().mean()) - 0.5) < 5 * 0.5 / 512 ** 0.5
    # the same activations, by the same number
    assert torch.equal(first[1], second[1]) and (first[1] == 0).any()
    # a run of one process goes on from the first rank's state as that rank does
    layer = tb.DropoutAdd(0.5)
    layer.load_state_dict(state)
    assert torch.equal(layer(torch.ones(16, 32)), first[0])


def test_replicas_of_a_generator():
    rng = torch.tensor([(1 << 62) + 12345, 7])
    first = tb.rng_next(rng.clone())
    assert torch.equal(first, rng) and torch.equal(tb.rng_next(rng.clone(), 0), rng)
    masks = []
    for replica in (0, 1, 2, 255, -1):
        state = rng.clone()
        taken = tb.rng_next(state, replica)
        assert int(taken[0]) % (1 << 64) == (int(rng[0]) + replica * 0x9E3779B97F4A7C15) % (1 << 64)
        assert int(taken[1]) == 7 and int(state[1]) == 8 and int(state[0]) == int(rng[0])
        masks.append(dropout_mask(taken, 64, 256, 0.5))
    for i, a in enumerate(masks):
        for b in masks[:i]:
            assert abs(float((a == b).float().mean()) - 0.5) < 5 * 0.5 / a.numel() ** 0.5


def test_a_copy_with_a_seed_of_its_own():
    x = torch.ones(8, 64)
    layer = tb.DropoutAdd(0.5)
    twin = copy.deepcopy(layer)
    assert torch.equal(layer(x), twin(x))
    twin.reseed()
    assert not torch.equal(layer(x), twin(x))
    twin.reseed(5)
    assert twin.rng.tolist() == [5, 0]


@pytest.mark.parametrize("reentrant", [False, True])
def test_a_call_that_is_run_again_drops_what_it_dropped(reentrant):
    layer = tb.DropoutAdd(0.5)
    x = torch.ones(16, 64, requires_grad=True)
    y = checkpoint(layer, x, use_reentrant=reentrant)
    y.sum().backward()
    # (ones through the same mask, both ways)
    assert torch.equal(x.grad, y.detach())
    assert int(layer.rng[1]) == 1


@pytest.mark.parametrize("reentrant", [False, True])
def test_recomputed_blocks_give_the_gradients_of_kept_ones(reentrant):
    torch.manual_seed(0)
    blocks = torch.nn.ModuleList(torch.nn.Sequential(torch.nn.Linear(24, 24), tb.DropoutAdd(0.3), torch.nn.Tanh(), torch.nn.Linear(24, 24))
                                 for _ in range(3))
    shared = tb.DropoutAdd(0.2)     # called once a block and batch
    x = torch.randn(5, 24)

    def block(i, v):
        return shared(blocks[i](v), v)

    def step(again):
        leaf = x.clone().requires_grad_()
        outs = []
        for scale in (1.0, 2.0):    # two batches in front of the backward pass
            v = leaf * scale
            for i in range(3):
                v = checkpoint(block, i, v, use_reentrant=reentrant) if again else block(i, v)
            outs.append(v)
        total = outs[0].sum() + (outs[1] ** 2).sum()
        blocks.zero_grad()
        total.backward()
        return [total.detach(), leaf.grad, *(p.grad.clone() for p in blocks.parameters())]

    state = {k: v.clone() for k, v in blocks.state_dict().items()}, shared.rng.clone()
    kept = step(False)
    blocks.load_state_dict(state[0])
    shared.rng.copy_(state[1])
    for a, b in zip(kept, step(True)):
        assert torch.allclose(a, b, rtol=1e-6, atol=1e-7)
    assert int(shared.rng[1]) == int(state[1][1]) + 6


def test_a_call_run_twice_again_and_calls_in_any_order():
    layer = tb.DropoutAdd(0.5)
    x = torch.ones(8, 64, requires_grad=True)
    ys = [checkpoint(layer, x, use_reentrant=False) for _ in range(3)]
    assert not torch.equal(ys[0], ys[1])
    for k in (1, 1, 0, 2, 1):
        dx, = torch.autograd.grad(ys[k], x, torch.ones_like(x), retain_graph=True)
        assert torch.equal(dx, ys[k].detach())
    assert int(layer.rng[1]) == 3


def test_a_call_run_again_without_its_generator_is_refused():
    layer = tb.DropoutAdd(0.5)
    x = torch.ones(8, 64, requires_grad=True)
    y = checkpoint(torch.nn.Sequential(layer, torch.nn.Tanh()), x, use_reentrant=False, preserve_rng_state=False)
    torch.rand(1)
    with pytest.raises(RuntimeError, match="preserve_rng_state"):
        y.sum().backward()


def test_ordinary_calls_draw_nothing_from_pytorch():
    layer = tb.DropoutAdd(0.5)
    torch.manual_seed(3)
    want = torch.rand(4)
    torch.manual_seed(3)
    layer(torch.ones(4, 4, requires_grad=True)).sum().backward()
    assert torch.equal(torch.rand(4), want)


def test_bfloat16_is_rounded_once():
    """As in the device's kernels: product, sum and norm in float."""
    gen = torch.Generator().manual_seed(0)
    x, r = (torch.randn(40, 70, generator=gen).bfloat16() for _ in range(2))
    w, b = torch.randn(2, 70, generator=gen)
    rng, p = torch.tensor([3, 4]), 0.1
    keep = dropout_mask(rng, 40, 70, p)
    want = r.double() + keep * x.double() * (65536 / (65536 - round(65536 * p)))
    assert torch.equal(tb.dropout_add(x, rng, p, r), want.float().bfloat16())
    y, total = tb.dropout_add_layer_norm(x, rng, p, r, w, b)
    assert y.dtype == total.dtype == torch.bfloat16
    assert torch.equal(total, want.float().bfloat16())
    norm = torch.nn.functional.layer_norm(want, (70,), w.double(), b.double())
    # one rounding to eight bits (seven behind the leading one: half of 2^-7), and 2^-20 of float beside it
    assert ((y.double() - norm).abs() <= (2.0 ** -8 + 2.0 ** -20) * norm.abs() + 2.0 ** -20).all()


def test_a_probability_without_a_generator_is_refused():
    with pytest.raises(RuntimeError, match="needs rng"):
        tb.dropout_add(torch.ones(3, 4), None, 0.5)
    assert torch.equal(tb.dropout_add(torch.ones(3, 4), None, 0.0), torch.ones(3, 4))
