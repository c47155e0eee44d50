"""Sampling from logits against its definition in 64 bits: tokens have to be equal.  (Weights are off by 2^-45 each on the device: a random
number would have to meet a border between two tokens to some 2^-36.)"""
import math

import numpy as np
import pytest
import torch

import butterfly_amd as tb

pytestmark = pytest.mark.gpu


def one_row(row, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    row = np.where(np.isnan(row), -np.inf, row) + 0.0
    if row.max() == -np.inf:
        return -1
    if not temperature > 0:
        return int(row.argmax())
    ranked = np.argsort(-row, kind="stable")
    if top_k > 0:
        ranked = ranked[:top_k]
    x = row[ranked]
    with np.errstate(invalid="ignore"):
        p = np.where(x == x[0], 1.0, np.exp((x - x[0]) / temperature))
    p = np.where(x == -np.inf, 0.0, p)
    ranked, p = ranked[p > 0], p[p > 0]
    if top_p < 1:
        running = np.cumsum(p)
        number = 1 + np.searchsorted(running[:-1], max(top_p, 0.0) * running[-1], side="left")
        ranked, p = ranked[:number], p[:number]
    ranked, p = ranked[p >= min(min_p, 1.0)], p[p >= min(min_p, 1.0)]
    by_index = np.argsort(ranked)
    ranked, running = ranked[by_index], np.cumsum(p[by_index])
    return int(ranked[min(np.searchsorted(running, u * running[-1], side="right"), len(ranked) - 1)])


def check(logits, uniform, **settings):
    got = tb.sample(logits.cuda(), uniform.cuda(), **{k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in settings.items()})
    assert got.dtype == torch.int64 and got.shape == logits.shape[:-1]
    host = tb.sample(logits, uniform, **settings)
    rows, us = logits.double().reshape(-1, logits.shape[-1]).numpy(), uniform.double().reshape(-1).numpy()
    each = {k: v.double().reshape(-1).numpy() if isinstance(v, torch.Tensor) and k != "top_k" else v.reshape(-1).numpy() if isinstance(v, torch.Tensor)
            else [v] * len(rows) for k, v in settings.items()}
    want = [one_row(rows[i], us[i], **{k: v[i] for k, v in each.items()}) for i in range(len(rows))]
    assert got.reshape(-1).tolist() == want
    assert host.reshape(-1).tolist() == want


FILTERS = [{}, {"temperature": 0.7}, {"top_k": 1}, {"top_k": 40}, {"top_p": 0.9}, {"top_p": 0.01}, {"min_p": 0.05}, {"temperature": 1.7, "top_k": 100, "top_p": 0.8, "min_p": 0.02},
           {"top_k": 400, "top_p": 0.999}, {"temperature": 0.0}, {"temperature": 100.0, "top_p": 0.5}, {"temperature": 0.01, "top_p": 0.9}]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("filters", FILTERS)
@pytest.mark.parametrize("entries", [1, 5, 64, 1000, 4097, 30001])
def test_filters(entries, filters, dtype):
    gen = torch.Generator().manual_seed(entries)
    logits = (torch.randn(7, entries, generator=gen) * 3).to(dtype)
    check(logits, torch.rand(7, generator=gen), **filters)


@pytest.mark.parametrize("dtype, entries", [(torch.float32, 70000), (torch.bfloat16, 140001), (torch.float32, 1 << 17), (torch.bfloat16, 1 << 17), (torch.bfloat16, 1 << 19)])
def test_large_vocabularies(dtype, entries):
    gen = torch.Generator().manual_seed(entries)
    logits = (torch.randn(3, entries, generator=gen) * 2).to(dtype)
    for filters in ({}, {"top_p": 0.9}, {"top_k": 50, "top_p": 0.9, "min_p": 0.01}, {"temperature": 0.0}):
        check(logits, torch.rand(3, generator=gen), **filters)


def test_settings_of_each_row():
    gen = torch.Generator().manual_seed(3)
    logits = torch.randn(4, 5, 777, generator=gen) * 2
    shape = (4, 5)
    temperature = torch.rand(shape, generator=gen) + 0.3
    temperature[1, 2] = 0.0
    check(logits, torch.rand(shape, generator=gen), temperature=temperature, top_k=torch.randint(-1, 60, shape, generator=gen),
          top_p=torch.rand(shape, generator=gen) * 1.2, min_p=torch.rand(shape, generator=gen) * 0.1 - 0.02)
    check(logits[0, 0], torch.rand((), generator=gen), top_p=0.7)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_ties(dtype):
    equal = torch.zeros(4, 1000, dtype=dtype)
    u = torch.tensor([0.0, 0.25, 0.5, 0.999])
    for filters in ({}, {"top_k": 10}, {"top_p": 0.5}, {"top_k": 100, "top_p": 0.5}, {"min_p": 1.0}, {"temperature": 0.0}):
        check(equal, u, **filters)
    # few distinct values, the border inside one of them
    steps = torch.randint(-3, 4, (40, 2000), generator=torch.Generator().manual_seed(0)).to(dtype)
    u = torch.rand(40, generator=torch.Generator().manual_seed(1))
    for filters in ({"top_k": 300}, {"top_p": 0.5}, {"top_k": 700, "top_p": 0.6, "min_p": 0.1}, {"top_p": 0.9, "min_p": 0.4}):
        check(steps, u, **filters)
    signed = torch.tensor([[0.0, -0.0, 0.0, -0.0, -1.0]], dtype=dtype)
    for k in range(1, 5):
        check(signed, torch.tensor([0.99]), top_k=k)
    check(signed, torch.tensor([0.5]), temperature=0.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_masked_and_not_finite(dtype):
    gen = torch.Generator().manual_seed(5)
    logits = (torch.randn(8, 3001, generator=gen) * 2).to(dtype)
    u = torch.rand(8, generator=gen)
    logits[0] = -math.inf                       # nothing left
    logits[1, 1:] = -math.inf                   # one left
    logits[2, torch.rand(3001, generator=gen) < 0.9] = -math.inf
    logits[3, torch.rand(3001, generator=gen) < 0.9] = torch.finfo(dtype).min
    logits[4, torch.rand(3001, generator=gen) < 0.5] = math.nan
    logits[5, [17, 2000]] = math.inf
    logits[6] = math.nan
    logits[7, :] = torch.finfo(dtype).max
    for filters in ({}, {"top_k": 5}, {"top_p": 0.7}, {"min_p": 0.1}, {"temperature": 0.0}, {"top_k": 2000, "top_p": 0.95, "min_p": 0.001}):
        check(logits, u, **filters)
    # more to be kept than there is
    check(logits[1:3], u[:2], top_k=400)


@pytest.mark.parametrize("spread, shift", [(1e-3, 0.0), (1e-3, 1000.0), (30.0, 0.0), (1e4, -1e6), (1e-30, 0.0)])
def test_values_of_all_sizes(spread, shift):
    gen = torch.Generator().manual_seed(9)
    logits = torch.randn(6, 5000, generator=gen) * spread + shift
    for filters in ({"top_p": 0.8}, {"top_k": 33, "top_p": 0.9}, {"temperature": spread, "top_p": 0.8}, {"temperature": spread, "top_k": 1000}):
        check(logits, torch.rand(6, generator=gen), **filters)


def test_random_numbers_at_the_ends():
    logits = torch.randn(3, 500)
    for u in (0.0, 1.0 - 2.0 ** -24):
        for filters in ({}, {"top_k": 3}, {"top_p": 0.5}):
            check(logits, torch.full((3,), u), **filters)
    last = tb.sample(logits.cuda(), torch.tensor([1.0, 2.0, -1.0], device="cuda"))
    assert last.tolist() == [499, 499, 0]


def test_frequencies_of_the_tokens():
    """Evenly spread numbers give every token its share, to a number or two."""
    logits = torch.tensor([0.0, 1.0, -1.0, 2.0, 0.5])
    n = 10000
    tokens = tb.sample(logits.expand(n, 5).cuda(), ((torch.arange(n) + 0.5) / n).cuda(), temperature=0.8)
    counts = torch.bincount(tokens.cpu(), minlength=5)
    assert float((counts / n - torch.softmax(logits / 0.8, 0)).abs().max()) < 2.0 / n


def test_strides_streams_and_capture():
    gen = torch.Generator().manual_seed(2)
    wide = torch.randn(6, 2003, generator=gen).cuda()
    u = torch.rand(6, generator=gen).cuda()
    want = tb.sample(wide[:, 1:2002].contiguous(), u, top_p=0.8)
    assert torch.equal(tb.sample(wide[:, 1:2002], u, top_p=0.8), want)
    assert torch.equal(tb.sample(wide.t().contiguous().t()[:, 1:2002], u, top_p=0.8), want)
    assert torch.equal(tb.sample(wide[::2, 1:2002], u[::2], top_p=0.8), want[::2])
    assert torch.equal(tb.sample(wide[:1, 1:2002].expand(6, 2001), u[:1].expand(6), top_p=0.8), want[:1].expand(6))
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = tb.sample(wide[:, 1:2002], u, top_p=0.8)
    stream.synchronize()
    assert torch.equal(other, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        token = tb.sample(wide, u, top_k=40, top_p=0.9)
    for _ in range(3):
        u.copy_(torch.rand(6, generator=gen))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(token, tb.sample(wide, u, top_k=40, top_p=0.9))


def test_refusals():
    x, u = torch.zeros(2, 5, device="cuda"), torch.zeros(2, device="cuda")
    assert tb.sample(x[:0], u[:0]).shape == (0,)
    for text, call in (("float32 and bfloat16", lambda: tb.sample(x.double(), u)), ("uniform must have the shape", lambda: tb.sample(x, u[:1])),
                       ("uniform must be", lambda: tb.sample(x, u.double())), ("top_k must be", lambda: tb.sample(x, u, top_k=u)),
                       ("temperature must have", lambda: tb.sample(x, u, temperature=u[:1])), ("on the device", lambda: tb.sample(x, u.cpu())),
                       ("shape", lambda: tb.sample(x[:, :0], u)), ("2\\^19", lambda: tb.sample(torch.zeros(1, (1 << 19) + 1, device="cuda"), u[:1]))):
        with pytest.raises(RuntimeError, match=text):
            call()


def test_settings_at_their_ends():
    logits = torch.tensor([[0.0, 1.0, 3.0, 2.0]] * 4)
    u = torch.tensor([0.01, 0.3, 0.6, 0.99])
    for filters in ({"min_p": math.nan}, {"top_p": math.nan}, {"temperature": math.nan}, {"temperature": 1e-300}, {"temperature": 1e-38},
                    {"temperature": math.inf}, {"temperature": 1e30, "top_p": 0.6}, {"temperature": 1e-40, "top_p": 0.5, "min_p": 0.1},
                    {"temperature": -math.inf}, {"top_k": 1 << 62}, {"top_k": -(1 << 62)}, {"top_p": -1.0}, {"min_p": math.inf}):
        assert tb.sample(logits.cuda(), u.cuda(), **filters).tolist() == tb.sample(logits, u, **filters).tolist(), filters


def test_a_row_without_more():
    """Logits of one dimension, a random number of none."""
    logits = torch.randn(77, generator=torch.Generator().manual_seed(3))
    token = tb.sample(logits.cuda(), torch.tensor(0.7, device="cuda"), top_k=torch.tensor(9, device="cuda"))
    assert token.shape == () and int(token) == int(tb.sample(logits, torch.tensor(0.7), top_k=9))
