"""Dropout modules in several processes and as copies, on the host."""
import copy
import os
import tempfile

import torch
import torch.distributed as dist
import torch.multiprocessing as mp

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
