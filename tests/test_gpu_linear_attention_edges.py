"""Linear attention: decays that are not finite, bits that results keep.  References are the definition in 64 bits, step by step, with
gradients by automatic differentiation; tolerances as for any other call (float32 1e-5 of the largest; bfloat16 results
rounded once, what they are summed from has 16 bits: 2^-8 + 2^-12)."""
import math

import pytest
import torch

import butterfly_amd as tb

pytestmark = pytest.mark.gpu

NAMES = ("q", "k", "v", "log_decay", "state")
RESULTS = ("o", "last", "d_q", "d_k", "d_v", "d_log_decay", "d_state")


def make(batch, steps, heads, groups, features, values, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed + 1000 * steps + 10 * features + values)

    def randn(*shape, dtype=dtype):
        return torch.randn(*shape, generator=gen).to(dtype)

    return {"q": randn(batch, steps, groups, features), "k": randn(batch, steps, groups, features), "v": randn(batch, steps, heads, values),
            "log_decay": -torch.rand(batch, steps, heads, generator=gen) * 0.05, "state": randn(batch, heads, features, values, dtype=torch.float32),
            "grad": randn(batch, steps, heads, values), "grad_last": randn(batch, heads, features, values, dtype=torch.float32)}


def definition(v, scale, reset=None):
    leaves = {k: v[k].double().requires_grad_() for k in NAMES}
    shared = v["v"].shape[2] // v["q"].shape[2]
    q, k = (leaves[n].repeat_interleave(shared, 2) for n in "qk")
    log_decay = leaves["log_decay"]
    if reset is not None:
        # (the decay of a reset step meets nothing)
        log_decay = torch.where(reset.unsqueeze(-1), 0.0, log_decay)
    s, out = leaves["state"], []
    for t in range(v["v"].shape[1]):
        decayed = torch.exp(log_decay[:, t])[..., None, None] * s
        if reset is not None and bool(reset[:, t].any()):
            assert bool(reset[:, t].all())
            decayed = torch.zeros_like(s)
        s = decayed + k[:, t, :, :, None] * leaves["v"][:, t, :, None, :]
        out.append(scale * (q[:, t].unsqueeze(-1) * s).sum(-2))
    o = torch.stack(out, 1)
    d = torch.autograd.grad([o, s], list(leaves.values()), [v["grad"].double(), v["grad_last"].double()])
    return dict(zip(RESULTS, (o.detach(), s.detach(), *d)))


def device(v, scale, reset=None):
    leaves = [v[k].cuda().requires_grad_() for k in NAMES]
    o, last = tb.linear_attention(*leaves, None if reset is None else reset.cuda(), scale)
    d = torch.autograd.grad([o, last], leaves, [v["grad"].cuda(), v["grad_last"].cuda()])
    return {k: t.detach().cpu().double() for k, t in zip(RESULTS, (o, last, *d))}


@pytest.mark.parametrize("bad", [math.nan, math.inf, 1e30])
@pytest.mark.parametrize("dtype, size", [(torch.float32, 20), (torch.bfloat16, 20), (torch.float32, 100), (torch.bfloat16, 100)])
@pytest.mark.parametrize("at, resets", [((90,), ()), ((64,), ()), ((95,), ()), ((0,), ()), ((70, 80), ()), ((90,), (80, 100)), ((80,), (80,)), ((100, 250), (70, 200))])
def test_decays_that_are_not_finite(at, resets, dtype, size, bad):
    """What a bad decay has no part in, its own chunk's later steps among them, is as it is without it: outputs and queries' gradients of
    earlier steps, values' and keys' gradients of that step and the later ones, other documents, other heads."""
    v = make(1, 300, 2, 1, size, size + 4, dtype)
    reset = None
    if resets:
        reset = torch.zeros(1, 300, dtype=torch.bool)
        reset[:, list(resets)] = True
    v["log_decay"][0, list(at), 0] = bad
    want, got = definition(v, 0.2, reset), device(v, 0.2, reset)
    for name in RESULTS:
        if name == "d_log_decay":
            continue
        there = torch.isfinite(want[name])
        assert torch.equal(torch.isfinite(got[name]), there), name
        if dtype == torch.float32 or name in ("last", "d_state"):
            tol = 1e-5
        else:
            tol = 2.0 ** -8 + 2.0 ** -12
        w, g = want[name][there], got[name][there]
        # (queries and keys are shared by both heads: a sum of two)
        assert w.numel() == 0 or float((g - w).abs().max() / w.abs().max()) <= tol, name
    # decays' gradients: not finite where they are not, and all of that document's in the chunk
    assert not bool((torch.isfinite(got["d_log_decay"]) & ~torch.isfinite(want["d_log_decay"])).any())
    assert bool(torch.isfinite(got["d_log_decay"][..., 1]).all())


@pytest.mark.parametrize("shape", [(2, 200, 4, 2, 64, 64), (2, 97, 2, 1, 128, 128), (1, 300, 6, 2, 100, 100), (1, 700, 2, 1, 128, 72), (1, 1000, 2, 2, 64, 64), (1, 129, 3, 3, 17, 33)])
def test_bfloat16_keeps_the_bits_that_it_says(shape):
    """Decays' gradients are floats and so is all that they are summed from: sums of products of bfloat16 numbers, which are exact,
    states and their gradients as three numbers (24 bits), decays; 1e-5 as with float32 inputs.  Results are rounded once (2^-8);
    inner factors, states and their gradients are read with 16 bits, wide heads' too: 2^-8 + 2^-12."""
    v = make(*shape, torch.bfloat16)
    want, got = definition(v, shape[4] ** -0.5), device(v, shape[4] ** -0.5)
    for name in RESULTS:
        err = float((got[name] - want[name]).abs().max() / want[name].abs().max())
        assert err <= (1e-5 if name in ("last", "d_state", "d_log_decay") else 2.0 ** -8 + 2.0 ** -12), (name, err)
