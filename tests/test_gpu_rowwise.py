"""Layer norm, dropout with residual, and both in one, against the formulas in 64 bits.

Errors are max |error| / max |reference| of a tensor.  float32: a row's statistics are sums of at most some 60 roundings
one after another (columns a lane holds, lanes, wavefronts), a column sum over R rows of R / slices + slices, all of 2^-24,
with room for cancellation between the three terms of the input's gradient: 1e-5.  bfloat16: results are
rounded once (2^-9 of their own magnitude), and a backward pass behind a sum starts from that sum
rounded (2^-9 again, in every factor of a column sum): 2^-7."""
import numpy as np
import pytest
import torch

import butterfly_amd as tb
from butterfly_amd.rowwise import dropout_mask

pytestmark = pytest.mark.gpu

TOL = {torch.float32: 1e-5, torch.bfloat16: 2.0 ** -7}
DTYPES = [torch.float32, torch.bfloat16]


def randn(*shape, dtype=torch.float32, seed=0, scale=1.0, shift=0.0):
    gen = torch.Generator().manual_seed(seed + sum(shape))
    return (torch.randn(*shape, generator=gen) * scale + shift).to(dtype).cuda()


def err(a, b):
    a, b = a.detach().double().cpu(), b.detach().double().cpu()
    assert a.shape == b.shape
    if b.numel() == 0:
        return 0.0
    return float((a - b).abs().max() / b.abs().max().clamp(min=1e-30))


def reference(x, g, residual=None, keep=None, p=0.0, weight=None, bias=None, eps=1e-5, g_sum=None, norm=True):
    """Outputs and gradients from the formulas, in 64 bits on the host."""
    wide = lambda t: None if t is None else t.detach().double().cpu()  # noqa: E731
    x, g, residual, weight, bias, g_sum = (wide(t) for t in (x, g, residual, weight, bias, g_sum))
    threshold = round(65536 * p)
    factor = 1.0
    if threshold:
        factor = keep.cpu().double() * (65536 / (65536 - threshold) if threshold < 65536 else 0.0)
    total = x * factor + (0 if residual is None else residual)
    out = {"sum": total, "y": total}
    d = g
    if norm:
        mean = total.mean(-1, keepdim=True)
        r = 1 / torch.sqrt(((total - mean) ** 2).mean(-1, keepdim=True) + eps)
        u = (total - mean) * r
        out["y"] = u * (1 if weight is None else weight) + (0 if bias is None else bias)
        lead = tuple(range(g.dim() - 1))
        out["d_weight"], out["d_bias"] = (g * u).sum(lead), g.sum(lead)
        gw = g * (1 if weight is None else weight)
        d = r * (gw - gw.mean(-1, keepdim=True) - u * (gw * u).mean(-1, keepdim=True)) + (0 if g_sum is None else g_sum)
    out["d_residual"], out["d_x"] = d, d * factor
    return out


COLS = [1, 2, 7, 8, 63, 64, 65, 128, 200, 257, 512, 513, 1000, 1024, 1500, 2048, 2049, 4096, 5000, 8192, 9001, 16384, 16385, 20001]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", COLS)
def test_layer_norm_and_gradients(cols, dtype):
    for rows in (1, 3, 70) + ((517,) if cols <= 2048 else ()):
        x = randn(rows, cols, dtype=dtype, seed=1, shift=0.5).requires_grad_()
        w = randn(cols, dtype=dtype, seed=2, scale=0.3, shift=1.0).requires_grad_()
        b = randn(cols, dtype=dtype, seed=3).requires_grad_()
        g = randn(rows, cols, dtype=dtype, seed=4)
        y = tb.layer_norm(x, w, b, 1e-3)
        grads = torch.autograd.grad(y, (x, w, b), g)
        ref = reference(x, g, weight=w, bias=b, eps=1e-3)
        assert y.dtype == dtype and [t.dtype for t in grads] == [dtype] * 3
        # (of one column the gradient is zero, of two zero but for eps / (var + eps), since u is +-1 whatever x is: the
        # difference of terms that cancel is held to the size of its terms)
        assert err(y, ref["y"]) < TOL[dtype]
        scale = g.double().abs().max() * w.double().abs().max() / np.sqrt(1e-3) if cols <= 2 else ref["d_x"].abs().max()
        assert float((grads[0].detach().double().cpu() - ref["d_x"]).abs().max() / scale) < TOL[dtype], rows
        if cols > 1:
            assert err(grads[1], ref["d_weight"]) < TOL[dtype], rows
        assert err(grads[2], ref["d_bias"]) < TOL[dtype], rows


@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_norm_parameters_in_other_forms(dtype):
    x, g = randn(2, 33, 300, dtype=dtype, seed=5).requires_grad_(), randn(2, 33, 300, dtype=dtype, seed=6)
    for weight, bias in ((None, None), (randn(300, seed=7), None), (None, randn(300, seed=8)), (randn(300, seed=7), randn(300, seed=8))):
        params = [t.requires_grad_() for t in (weight, bias) if t is not None]
        y = tb.layer_norm(x, weight, bias)
        grads = torch.autograd.grad(y, [x] + params, g)
        ref = reference(x, g, weight=weight, bias=bias)
        assert err(y, ref["y"]) < TOL[dtype] and err(grads[0], ref["d_x"]) < TOL[dtype]
        for t, got in zip(params, grads[1:]):
            assert got.dtype == torch.float32
            assert err(got, ref["d_weight" if t is weight else "d_bias"]) < 1e-5


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cols", [40, 300, 1000, 3000])
def test_rows_with_other_strides_and_alignments(cols, dtype):
    base = randn(50, cols + 37, dtype=dtype, seed=9)
    g = randn(50, cols, dtype=dtype, seed=10)
    w, b = randn(cols + 1, dtype=dtype, seed=11)[1:], randn(cols + 3, dtype=dtype, seed=12)[3:]
    views = {
        "odd offset": base[:, 5:5 + cols],
        "every other row": base[::2, 3:3 + cols],
        "transposed": randn(cols, 50, dtype=dtype, seed=13).t(),
        "one row for all": base[:1, 1:1 + cols].expand(50, cols),
        "three dimensions": randn(5, 10, cols, dtype=dtype, seed=14).transpose(0, 1),
    }
    for name, x in views.items():
        gv = g[:x.shape[0]] if x.dim() == 2 else randn(10, 5, cols, dtype=dtype, seed=15)
        x = x.detach().requires_grad_()
        for grad in (gv, torch.ones((), dtype=dtype, device="cuda").expand(gv.shape), gv.flip(0).contiguous().flip(0)):
            y = tb.layer_norm(x, w, b)
            ref = reference(x, grad, weight=w, bias=b)
            assert err(y, ref["y"]) < TOL[dtype], name
            dx, = torch.autograd.grad(y, x, grad)
            scale = float(w.double().abs().max() * grad.double().abs().max() / x.double().std())
            assert float((dx.double().cpu() - ref["d_x"]).abs().max()) < TOL[dtype] * max(scale, float(ref["d_x"].abs().max())), name


def test_large_offsets_small_spread_and_constant_rows():
    # the deviations are formed from the row's own mean: with an offset of 1000 the inputs' own rounding (2^-14) remains
    for cols in (100, 1000, 3000, 20000):
        x = randn(8, cols, seed=20) + 1000.0
        ref = reference(x, x)
        assert err(tb.layer_norm(x), ref["y"]) < 1e-5
        c = torch.full((3, cols), 7.25, device="cuda")
        b = randn(cols, seed=21)
        assert torch.equal(tb.layer_norm(c, None, b), b.expand(3, cols))


@pytest.mark.parametrize("cols", [64, 700, 4000, 17000])
def test_a_row_that_is_not_finite_stays_alone(cols):
    x, g = randn(40, cols, seed=22), randn(40, cols, seed=23)
    clean = tb.layer_norm(x)
    x2 = x.clone()
    x2[7, cols // 2], x2[11, 0] = float("nan"), float("inf")
    x2.requires_grad_()
    y = tb.layer_norm(x2)
    dx, = torch.autograd.grad(y, x2, g)
    others = [i for i in range(40) if i not in (7, 11)]
    assert torch.equal(y[others], clean[others]) and torch.isfinite(dx[others]).all()
    assert torch.isnan(y[7]).all() and torch.isnan(y[11]).all()


def test_empty_tensors():
    w = torch.ones(5, device="cuda", requires_grad=True)
    x = torch.empty(0, 5, device="cuda", requires_grad=True)
    y = tb.layer_norm(x, w)
    assert y.shape == (0, 5)
    dx, dw = torch.autograd.grad(y, (x, w), torch.empty(0, 5, device="cuda"))
    assert dx.shape == (0, 5) and torch.equal(dw, torch.zeros(5, device="cuda"))
    assert tb.layer_norm(torch.empty(3, 0, device="cuda")).shape == (3, 0)
    assert tb.dropout_add(torch.empty(0, device="cuda"), None, 0.0).shape == (0,)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (5, 8), (70, 33), (9, 64), (300, 784), (17, 1000), (4, 2049), (2, 9000), (2, 3, 40)])
@pytest.mark.parametrize("p", [0.1, 0.5])
def test_dropout_add(shape, p, dtype):
    # (a seed and a call number with bits in all four words of key and counter, the sign bits among them)
    rng = torch.tensor([-0x123456789ABCDEF, 0x7FEDCBA987654321], device="cuda")
    rows, cols = int(np.prod(shape[:-1])), shape[-1]
    keep = dropout_mask(rng.cpu(), rows, cols, p).reshape(shape)
    x, r = randn(*shape, dtype=dtype, seed=30).requires_grad_(), randn(*shape, dtype=dtype, seed=31).requires_grad_()
    g = randn(*shape, dtype=dtype, seed=32)
    for residual in (None, r):
        y = tb.dropout_add(x, rng, p, residual)
        ref = reference(x, g, residual, keep, p, norm=False)
        # one product and one sum in float32, rounded once
        assert err(y, ref["y"]) < {torch.float32: 3e-7, torch.bfloat16: 2.0 ** -8}[dtype]
        assert residual is not None or torch.equal((y != 0).cpu(), keep & (x != 0).cpu())
        wanted = [x] if residual is None else [x, r]
        grads = torch.autograd.grad(y, wanted, g)
        assert err(grads[0], ref["d_x"]) < {torch.float32: 3e-7, torch.bfloat16: 2.0 ** -8}[dtype]
        assert torch.equal(grads[0] == 0, ~keep.cuda() | (g == 0))
        if residual is not None:
            assert torch.equal(grads[1], g)


def test_dropout_probabilities_at_the_ends():
    rng = torch.tensor([5, 6], device="cuda")
    x, r = randn(33, 100, seed=33), randn(33, 100, seed=34)
    assert torch.equal(tb.dropout_add(x, rng, 0.0), x)
    assert torch.equal(tb.dropout_add(x, None, 0.0, r), r + x)
    assert torch.equal(tb.dropout_add(x, rng, 1e-6, r), r + x)      # rounds to no 16-bit number at all
    assert torch.equal(tb.dropout_add(x, rng, 1.0, r), r)
    y, total = tb.dropout_add_layer_norm(x, rng, 1.0, r)
    assert torch.equal(total, r) and err(y, reference(r, r)["y"]) < 1e-5


def test_dropped_elements_are_zero_whatever_they_are():
    rng = torch.tensor([7, 8], device="cuda")
    keep = dropout_mask(rng, 20, 300, 0.5)
    x = torch.where(keep, randn(20, 300, seed=35), torch.tensor(float("nan"), device="cuda"))
    x[0] = torch.where(keep[0], x[0], torch.tensor(float("inf"), device="cuda"))
    assert torch.isfinite(tb.dropout_add(x, rng, 0.5)).all()
    x = x.requires_grad_()
    y, total = tb.dropout_add_layer_norm(x, rng, 0.5, None)
    assert torch.isfinite(y).all()
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    assert torch.isfinite(dx).all() and (dx[~keep] == 0).all()


def test_masks_of_other_calls_seeds_and_rows_are_others_and_their_shares_right():
    n = 1 << 20
    x = torch.ones(64, n // 64, device="cuda")
    masks = [tb.dropout_add(x, torch.tensor(k, device="cuda"), 0.25) != 0 for k in ((1, 0), (1, 1), (2, 0), (1 << 40, 0), (1, 1 << 40))]
    for i, a in enumerate(masks):
        # a share of n independent draws: five standard deviations
        assert abs(float(a.float().mean()) - 0.75) < 5 * (0.25 * 0.75 / n) ** 0.5
        for b in masks[:i]:
            assert abs(float((a == b).float().mean()) - 0.625) < 5 * (0.625 * 0.375 / n) ** 0.5
    assert abs(float((masks[0][1:] == masks[0][:-1]).float().mean()) - 0.625) < 5 * (0.625 * 0.375 / n) ** 0.5


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 5), (37, 64), (300, 100), (70, 513), (33, 1500), (20, 4096), (9, 8000), (5, 12001), (4, 18001)])
def test_dropout_add_layer_norm(shape, dtype):
    rng, p = torch.tensor([11, 12], device="cuda"), 0.2
    keep = dropout_mask(rng.cpu(), *shape, p)
    x, r = randn(*shape, dtype=dtype, seed=40).requires_grad_(), randn(*shape, dtype=dtype, seed=41, scale=2.0).requires_grad_()
    w, b = randn(shape[1], seed=42, scale=0.3, shift=1.0).requires_grad_(), randn(shape[1], seed=43).requires_grad_()
    g, gs = randn(*shape, dtype=dtype, seed=44), randn(*shape, dtype=dtype, seed=45)
    y, total = tb.dropout_add_layer_norm(x, rng, p, r, w, b)
    for wanted_sum in (gs, None):
        ref = reference(x, g, r, keep, p, w, b, g_sum=wanted_sum)
        outs, grads_in = ([y, total], [g, gs]) if wanted_sum is not None else ([y], [g])
        grads = torch.autograd.grad(outs, (x, r, w, b), grads_in, retain_graph=True)
        assert err(y, ref["y"]) < TOL[dtype] and err(total, ref["sum"]) < TOL[dtype]
        for got, name in zip(grads, ("d_x", "d_residual", "d_weight", "d_bias")):
            assert err(got, ref[name]) < TOL[dtype], name
        assert (grads[0][~keep.cuda()] == 0).all()
    # the sum's gradient alone
    dx, dr = torch.autograd.grad(total, (x, r), gs, retain_graph=True)
    assert torch.equal(dr, gs) and err(dx, reference(x, gs, r, keep, p, norm=False)["d_x"]) < TOL[dtype]
    # only some gradients asked for
    dw, = torch.autograd.grad(y, w, g)
    assert err(dw, ref["d_weight"]) < TOL[dtype]


def test_gradients_against_differences():
    """Central differences of <g, f> along random directions: with a step of 1/64 the third derivative's share (some
    1e-4) and the outputs' rounding (2^-24 sqrt(n) / step) both stay below 2e-3 of the derivative's scale."""
    rng, p, shape = torch.tensor([13, 14], device="cuda"), 0.3, (12, 200)
    args = [randn(*shape, seed=50), randn(*shape, seed=51), randn(200, seed=52, shift=1.0, scale=0.3), randn(200, seed=53)]
    g, gs = randn(*shape, seed=54), randn(*shape, seed=55)

    def value(a):
        y, total = tb.dropout_add_layer_norm(a[0], rng, p, a[1], a[2], a[3])
        return float((y.double() * g).sum() + (total.double() * gs).sum())

    leaves = [a.clone().requires_grad_() for a in args]
    y, total = tb.dropout_add_layer_norm(leaves[0], rng, p, leaves[1], leaves[2], leaves[3])
    grads = torch.autograd.grad((y, total), leaves, (g, gs))
    for k, grad in enumerate(grads):
        d = randn(*args[k].shape, seed=60 + k)
        h = 1 / 64
        up, down = list(args), list(args)
        up[k], down[k] = args[k] + h * d, args[k] - h * d
        numeric = (value(up) - value(down)) / (2 * h)
        scale = float(grad.double().norm() * d.double().norm())
        assert abs(numeric - float((grad.double() * d).sum())) < 2e-3 * scale, k


def test_same_bits_every_time_and_on_another_stream():
    rng = torch.tensor([15, 16], device="cuda")
    x, r, w, b = randn(3001, 1000, seed=70), randn(3001, 1000, seed=71), randn(1000, seed=72), randn(1000, seed=73)
    g = randn(3001, 1000, seed=74)
    leaves = [t.requires_grad_() for t in (x, r, w, b)]

    def step():
        y, total = tb.dropout_add_layer_norm(leaves[0], rng, 0.1, *leaves[1:])
        return [y, total, *torch.autograd.grad(y, leaves, g)]

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b_ in zip(first, again):
        assert torch.equal(a, b_)


def test_modules_draw_another_mask_a_call_and_none_in_eval():
    torch.manual_seed(0)
    drop, last = tb.DropoutAdd(0.5).cuda(), tb.DropoutAddLayerNorm(64, 0.5).cuda()
    x, r = randn(30, 64, seed=80), randn(30, 64, seed=81)
    before = drop.rng.clone()
    a, b = drop(x, r), drop(x, r)
    assert not torch.equal(a, b) and drop.rng.tolist() == [before[0].item(), before[1].item() + 2]
    assert torch.equal(a, tb.dropout_add(x, before, 0.5, r))
    # a state dict resumes the sequence of masks
    other = tb.DropoutAdd(0.5).cuda()
    other.load_state_dict(drop.state_dict())
    assert torch.equal(other(x, r), drop(x, r))
    assert not torch.equal(last(x, r)[0], last(x, r)[0])
    drop.eval(), last.eval()
    assert torch.equal(drop(x, r), r + x) and drop(x) is x
    assert torch.equal(last(x, r)[1], r + x)


def test_recorded_in_a_graph_every_replay_drops_others():
    torch.manual_seed(1)
    module = tb.DropoutAddLayerNorm(256, 0.5).cuda()
    x, g = randn(40, 256, seed=82), randn(40, 256, seed=83)
    step = tb.GraphedStep(lambda t: module(t)[0], x, g, params=tuple(module.parameters()))
    sums = []
    for _ in range(3):
        rng = module.rng.clone()
        y, grads = step(x, g)
        torch.cuda.synchronize()
        leaf = x.clone().requires_grad_()
        want, _ = tb.dropout_add_layer_norm(leaf, rng, 0.5, None, module.weight, module.bias)
        wanted = torch.autograd.grad(want, (leaf, module.weight, module.bias), g)
        assert torch.equal(y, want)
        for a, b in zip(grads, wanted):
            assert torch.equal(a, b)
        sums.append(float(y.sum()))
    assert len(set(sums)) == 3


def test_refusals():
    x, rng = randn(4, 8), torch.tensor([1, 2], device="cuda")
    for call in (
        lambda: tb.layer_norm(x.half()), lambda: tb.layer_norm(x, randn(7)), lambda: tb.layer_norm(x, randn(8).cpu()),
        lambda: tb.layer_norm(x, randn(8), randn(8, dtype=torch.bfloat16)), lambda: tb.layer_norm(x, eps=-1.0),
        lambda: tb.layer_norm(x, randn(8).double()), lambda: tb.layer_norm(torch.ones((), device="cuda")),
        lambda: tb.dropout_add(x, None, 0.5), lambda: tb.dropout_add(x, rng, 1.5), lambda: tb.dropout_add(x, rng, float("nan")),
        lambda: tb.dropout_add(x, rng.int(), 0.5), lambda: tb.dropout_add(x, rng[:1], 0.5), lambda: tb.dropout_add(x, rng.cpu(), 0.5),
        lambda: tb.dropout_add(x, rng, 0.5, randn(4, 7)), lambda: tb.dropout_add(x, rng, 0.5, randn(4, 8, dtype=torch.bfloat16)),
        lambda: torch.ops.torch_butterfly.layer_norm(x.cpu(), None, None, 1e-5), lambda: tb.DropoutAdd(1.5), lambda: tb.rng_next(rng[:1]),
    ):
        with pytest.raises((RuntimeError, ValueError)):
            call()
    leaf = x.clone().requires_grad_()
    y = tb.layer_norm(leaf)
    with torch.no_grad():
        leaf.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, leaf, torch.ones_like(y))
