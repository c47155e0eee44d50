"""The linear layer with softmax cross entropy against the definition in 64 bits.

Errors are max |error| / max |reference| of a tensor.  float32: a logit of magnitude l is off by some l 2^-20 (two factors of 22
bits, sums in float32), the probabilities by as much times l: 5e-5 at the logits of up to 16 used here.  bfloat16 (against
the definition at the bfloat16 inputs): the logits' gradient and the results are rounded to 2^-9 each: 2^-7.
The loss itself is float32 throughout: 1e-5 of 1 + its size."""
import pytest
import torch

import butterfly_amd as tb

pytestmark = pytest.mark.gpu

TOL = {torch.float32: 5e-5, torch.bfloat16: 2.0 ** -7}
DTYPES = [torch.float32, torch.bfloat16]


def make(rows, features, vocab, dtype, seed=0, ignored=0.2, scale=2.0):
    gen = torch.Generator(device="cuda").manual_seed(seed + rows + 7 * features + 11 * vocab)
    hidden = torch.randn(rows, features, device="cuda", generator=gen).to(dtype)
    weight = (torch.randn(vocab, features, device="cuda", generator=gen) * (scale / features ** 0.5)).to(dtype)
    target = torch.randint(0, vocab, (rows,), device="cuda", generator=gen)
    target[torch.rand(rows, device="cuda", generator=gen) < ignored] = -100
    if rows:
        target[0] = vocab - 1
    return hidden, weight, target


def reference(hidden, weight, target, grad, reduction, ignore=-100):
    h, w = hidden.detach().double(), weight.detach().double()
    counts = target != ignore
    n = int(counts.sum())
    hv, t = h[counts], target[counts]
    logits = hv @ w.t()
    lse = torch.logsumexp(logits, 1)
    each = torch.zeros(len(target), dtype=torch.float64, device="cuda")
    each[counts] = lse - logits.gather(1, t[:, None])[:, 0]
    g = torch.zeros(len(target), dtype=torch.float64, device="cuda")
    g[:] = grad.double() / (n if reduction == "mean" else 1)
    p = torch.exp(logits - lse[:, None])
    p.scatter_add_(1, t[:, None], torch.full((n, 1), -1.0, dtype=torch.float64, device="cuda"))
    p *= g[counts, None]
    dh = torch.zeros_like(h)
    dh[counts] = p @ w
    loss = each if reduction == "none" else each.sum() / (n if reduction == "mean" else 1)
    return loss, dh, p.t() @ hv


def err(a, b):
    assert a.shape == b.shape
    return float((a.detach().double() - b).abs().max() / b.abs().max().clamp(min=1e-30)) if b.numel() else 0.0


def check(hidden, weight, target, reduction="mean", ignore=-100, tol=None):
    h, w = hidden.detach().requires_grad_(), weight.detach().requires_grad_()
    gen = torch.Generator(device="cuda").manual_seed(5)
    grad = torch.randn(target.shape if reduction == "none" else (), device="cuda", generator=gen)
    loss = tb.linear_cross_entropy(h, w, target, ignore, reduction)
    assert loss.dtype == torch.float32
    dh, dw = torch.autograd.grad(loss, (h, w), grad)
    assert dh.dtype == h.dtype and dw.dtype == w.dtype
    want, want_h, want_w = reference(h, w, target, grad, reduction, ignore)
    assert (loss.double() - want).abs().max() <= 1e-5 * (1 + want.abs().max())
    tol = tol or TOL[h.dtype]
    assert err(dh, want_h) < tol and err(dw, want_w) < tol, (err(dh, want_h), err(dw, want_w))
    assert (dh[target == ignore] == 0).all()
    return loss, dh, dw


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [1, 2, 63, 64, 65, 128, 129, 257, 300])
def test_rows(rows, dtype):
    check(*make(rows, 96, 1000, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("features", [1, 2, 7, 8, 16, 63, 64, 65, 72, 100, 128, 129, 256, 520])
def test_features(features, dtype):
    check(*make(70, features, 500, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [1, 2, 3, 64, 127, 128, 129, 255, 256, 257, 1000, 5001])
def test_vocabularies(vocab, dtype):
    hidden, weight, target = make(90, 64, vocab, dtype)
    if vocab == 1:   # the only entry has probability one: losses and gradients are zero
        h, w = hidden.requires_grad_(), weight.requires_grad_()
        loss = tb.linear_cross_entropy(h, w, target)
        dh, dw = torch.autograd.grad(loss, (h, w))
        # (a logit of some 4 is off by 2^-20 of it at most)
        assert abs(float(loss)) < 1e-5 and dh.abs().max() < 1e-5 and dw.abs().max() < 1e-5
    else:
        check(hidden, weight, target)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
def test_reductions(reduction, dtype):
    check(*make(200, 80, 700, dtype), reduction)
    hidden, weight, target = make(200, 80, 700, dtype)
    check(hidden, weight, target.masked_fill(target == -100, 7), reduction, ignore=7)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,features,vocab", [(2048, 64, 16384), (3000, 1024, 4100), (16384, 32, 10000), (130, 2048, 9000), (5000, 24, 300)])
def test_large_tiles_pieces_and_split_sums(rows, features, vocab, dtype):
    """256 x 256 tiles in each of the three products; a vocabulary of several pieces; k steps in several parts."""
    check(*make(rows, features, vocab, dtype), "mean")
    check(*make(rows, features, vocab, dtype, seed=1), "none")


@pytest.mark.parametrize("dtype", DTYPES)
def test_leading_dimensions_and_strides(dtype):
    hidden, weight, target = make(60, 40, 300, dtype)
    loss, dh, dw = check(hidden, weight, target)
    cube = tb.linear_cross_entropy(hidden.view(3, 20, 40), weight, target.view(3, 20))
    assert torch.equal(cube, loss)
    assert tb.linear_cross_entropy(hidden.view(3, 20, 40), weight, target.view(3, 20), reduction="none").shape == (3, 20)
    assert tb.linear_cross_entropy(hidden[0], weight, target[0], reduction="none").shape == ()
    wide_h, wide_w = torch.zeros(60, 57, dtype=dtype, device="cuda"), torch.zeros(300, 64, dtype=dtype, device="cuda")
    wide_h[:, 3:43], wide_w[:, 8:48] = hidden, weight
    views = [(wide_h[:, 3:43], wide_w[:, 8:48]), (hidden.t().contiguous().t(), weight.t().contiguous().t()),
             (hidden, torch.cat((weight, weight))[::2].contiguous().repeat_interleave(2, 0)[::2])]
    assert torch.equal(tb.linear_cross_entropy(*views[0], target), loss)
    assert torch.equal(tb.linear_cross_entropy(*views[1], target), loss)
    check(*views[2], target)
    # one weight row for all entries: every entry is as likely, and the hidden rows' gradient sum_v p_v W_v - W_t is zero
    leaf = hidden.detach().requires_grad_()
    each = tb.linear_cross_entropy(leaf, weight[:1].expand(300, 40), target, reduction="none")
    assert (each[target != -100] - torch.log(torch.tensor(300.0))).abs().max() < 1e-5
    assert torch.autograd.grad(each.sum(), leaf)[0].abs().max() < TOL[dtype] * float(weight[0].abs().max())
    strided = torch.stack((target, target), 1)[:, 0]
    assert torch.equal(tb.linear_cross_entropy(hidden, weight, strided), loss)
    odd = torch.empty(300 * 40 + 1, dtype=dtype, device="cuda")[1:].view(300, 40).copy_(weight)
    assert torch.equal(tb.linear_cross_entropy(hidden, odd, target), loss)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
def test_ignored_rows_reach_nothing(reduction, dtype):
    hidden, weight, target = make(150, 64, 400, dtype, ignored=0.5)
    first = check(hidden, weight, target, reduction)
    bad = hidden.clone()
    bad[target == -100] = float("nan")
    bad[149 if int(target[149]) == -100 else int((target == -100).nonzero()[0])] = float("inf")
    for a, b in zip(first, check(bad, weight, target, reduction)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_all_rows_ignored_and_no_rows(dtype):
    hidden, weight, target = make(70, 64, 400, dtype)
    for t in (torch.full_like(target, -100), target[:0]):
        for reduction, value in (("mean", float("nan")), ("sum", 0.0)):
            h, w = hidden[:len(t)].detach().requires_grad_(), weight.detach().requires_grad_()
            loss = tb.linear_cross_entropy(h, w, t, reduction=reduction)
            assert torch.isnan(loss) if value != value else loss == value
            dh, dw = torch.autograd.grad(loss, (h, w))
            assert (dh == 0).all() and (dw == 0).all()
        h = hidden[:len(t)].detach().requires_grad_()
        each = tb.linear_cross_entropy(h, weight, t, reduction="none")
        assert torch.equal(each, torch.zeros(len(t), device="cuda"))
        assert (torch.autograd.grad(each, h, torch.ones_like(each))[0] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_targets_outside_the_vocabulary_make_nan(dtype):
    hidden, weight, target = make(40, 64, 300, dtype)
    for bad in (300, -1, 1 << 40):
        t = target.clone()
        t[5] = bad
        h, w = hidden.detach().requires_grad_(), weight.detach().requires_grad_()
        each = tb.linear_cross_entropy(h, w, t, reduction="none")
        assert torch.isnan(each[5]) and torch.isfinite(each[:5]).all() and torch.isfinite(each[6:]).all()
        dh, dw = torch.autograd.grad(each.sum(), (h, w))
        assert torch.isnan(dh[5]).all() and torch.isfinite(dh[:5]).all() and torch.isnan(dw).all()
        assert torch.isnan(tb.linear_cross_entropy(h, w, t))


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_logits(dtype):
    """Logits of some +-1000 (a softmax that is nearly one-hot): no overflow.  They are off by 1000 x 2^-20 (float32), so the
    probabilities that matter by some 1e-3."""
    hidden, weight, target = make(80, 64, 600, dtype, scale=400.0)
    h, w = hidden.requires_grad_(), weight.requires_grad_()
    grad = torch.ones((), device="cuda")
    loss = tb.linear_cross_entropy(h, w, target)
    want, want_h, want_w = reference(h, w, target, grad, "mean")
    assert abs(float(loss) - float(want)) < 1e-5 * (1 + abs(float(want)))
    dh, dw = torch.autograd.grad(loss, (h, w))
    assert err(dh, want_h) < max(2e-3, TOL[dtype]) and err(dw, want_w) < max(2e-3, TOL[dtype])


@pytest.mark.parametrize("up", [1e-25, 1e-6, 1e6, 1e25])
def test_float_operands_of_any_scale(up):
    hidden, weight, target = make(80, 100, 600, torch.float32)
    check(hidden * up, weight / up, target)


def test_float_rows_of_unlike_scale():
    """Numbers far below the operand's largest keep an absolute error of 2^-39 of that: rows 2^-12 of the others still have
    26 bits below them, so their own loss is as good as any."""
    hidden, weight, target = make(80, 100, 600, torch.float32)
    hidden[::2] *= 2.0 ** -12
    check(hidden, weight, target, "none")
    hidden, weight, target = make(80, 100, 600, torch.float32)
    weight[::2] *= 2.0 ** -12
    check(hidden, weight, target, "none")


@pytest.mark.parametrize("dtype", DTYPES)
def test_zeros_and_numbers_that_are_not_finite(dtype):
    hidden, weight, target = make(40, 64, 300, dtype, ignored=0.0)
    zero = tb.linear_cross_entropy(torch.zeros_like(hidden), weight, target, reduction="none")
    assert (zero - torch.log(torch.tensor(300.0))).abs().max() < 1e-5
    zero = tb.linear_cross_entropy(hidden, torch.zeros_like(weight), target, reduction="none")
    assert (zero - torch.log(torch.tensor(300.0))).abs().max() < 1e-5
    hidden[3, 5] = float("nan")
    each = tb.linear_cross_entropy(hidden, weight, target, reduction="none")
    assert torch.isnan(each[3])
    if dtype == torch.bfloat16:   # (float operands share one power of two, but a row's NaN stays its own)
        assert torch.isfinite(each[:3]).all() and torch.isfinite(each[4:]).all()
    weight[7, 1] = float("inf")
    assert not torch.isfinite(tb.linear_cross_entropy(hidden, weight, target))


def test_gradients_of_one_operand_alone_and_zero_upstream():
    hidden, weight, target = make(100, 64, 500, torch.float32)
    h, w = hidden.requires_grad_(), weight.requires_grad_()
    both = torch.autograd.grad(tb.linear_cross_entropy(h, w, target), (h, w))
    assert torch.equal(torch.autograd.grad(tb.linear_cross_entropy(h, w.detach(), target), h)[0], both[0])
    assert torch.equal(torch.autograd.grad(tb.linear_cross_entropy(h.detach(), w, target), w)[0], both[1])
    for reduction in ("mean", "none"):
        loss = tb.linear_cross_entropy(h, w, target, reduction=reduction)
        for d in torch.autograd.grad(loss, (h, w), torch.zeros_like(loss)):
            assert (d == 0).all()
    # shares of very unlike size
    g = torch.logspace(-6, 2, 100, device="cuda")
    each = tb.linear_cross_entropy(h, w, target, reduction="none")
    dh, dw = torch.autograd.grad(each, (h, w), g)
    _, want_h, want_w = reference(h, w, target, g, "none")
    assert err(dh, want_h) < 5e-5 and err(dw, want_w) < 5e-5


def test_gradients_against_differences():
    """Along random directions with a step of 1/64: the third derivative's share and the loss's rounding (2^-22 of it over the
    step) stay below 5e-3 of the derivative's scale."""
    hidden, weight, target = make(30, 40, 200, torch.float32)

    def value(h, w):
        return float(tb.linear_cross_entropy(h, w, target, reduction="none").double().sum())

    leaves = [hidden.clone().requires_grad_(), weight.clone().requires_grad_()]
    grads = torch.autograd.grad(tb.linear_cross_entropy(*leaves, target, reduction="sum"), leaves)
    for k, grad in enumerate(grads):
        d = torch.randn(leaves[k].shape, generator=torch.Generator().manual_seed(k)).cuda() / 4
        args = [hidden, weight]
        up, down = list(args), list(args)
        up[k], down[k] = args[k] + d / 64, args[k] - d / 64
        numeric = (value(*up) - value(*down)) * 32
        assert abs(numeric - float((grad.double() * d).sum())) < 5e-3 * float(grad.double().norm() * d.double().norm()), k


@pytest.mark.parametrize("dtype", DTYPES)
def test_same_bits_every_time_on_another_stream_and_in_a_graph(dtype):
    hidden, weight, target = make(300, 200, 3000, dtype)
    first = check(hidden, weight, target)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = check(hidden, weight, target)
    for a, b in zip(first, again):
        assert torch.equal(a, b)
    w = weight.detach().requires_grad_()
    grad = torch.ones((), device="cuda")
    step = tb.GraphedStep(lambda h: tb.linear_cross_entropy(h, w, target), hidden, grad, params=(w,))
    for k in range(3):
        h = (hidden * (1 + k)).requires_grad_()
        loss, grads = step(h.detach(), grad)
        torch.cuda.synchronize()
        want = tb.linear_cross_entropy(h, w, target)
        assert torch.equal(loss, want)
        for a, b in zip(grads, torch.autograd.grad(want, (h, w), grad)):
            assert torch.equal(a, b)


# ---- few rows (up to 64 and no more than features): kernels of their own ----

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,features,vocab", [
    (1, 1, 1), (1, 7, 33), (2, 2, 31), (3, 3, 5000), (5, 1000, 64), (15, 33, 32), (16, 31, 17), (17, 32, 15), (31, 127, 1001), (32, 2048, 300),
    (33, 129, 33001), (47, 64, 32768), (48, 520, 40003), (63, 65, 97), (64, 64, 2), (64, 1031, 36001), (7, 4096, 70000)])
def test_few_rows(rows, features, vocab, dtype):
    """Each number of 16-row tiles; vocabularies and features around the tiles of 16 and 32, the chunks of 32 and 64, the parts
    of 64 and 128 columns; vocabularies of both sizes of a workgroup's part (32768 on)."""
    for seed, reduction in enumerate(("mean", "none", "sum")):
        check(*make(rows, features, vocab, dtype, seed=seed), reduction)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,features,vocab", [(20, 75, 500), (50, 640, 33000)])
def test_few_rows_of_any_stride(rows, features, vocab, dtype):
    hidden, weight, target = make(rows, features, vocab, dtype)
    first = check(hidden, weight, target)
    wide = torch.full((rows, features + 13), float("nan"), dtype=dtype, device="cuda")
    wide[:, 5:5 + features] = hidden
    tall = torch.full((vocab, features + 11), float("nan"), dtype=dtype, device="cuda")
    tall[:, :features] = weight
    for a, b in zip(first, check(wide[:, 5:5 + features], tall[:, :features], target)):
        assert torch.equal(a, b)
    same = weight[:1].expand(vocab, features)
    each = tb.linear_cross_entropy(hidden, same, target, reduction="none")
    assert (each[target != -100] - torch.log(torch.tensor(float(vocab)))).abs().max() < 1e-5 * 12


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
def test_few_rows_ignored(reduction, dtype):
    hidden, weight, target = make(60, 64, 400, dtype, ignored=0.5)
    first = check(hidden, weight, target, reduction)
    bad = hidden.clone()
    bad[target == -100] = float("nan")
    for a, b in zip(first, check(bad, weight, target, reduction)):
        assert torch.equal(a, b)
    h, w = hidden.detach().requires_grad_(), weight.detach().requires_grad_()
    loss = tb.linear_cross_entropy(h, w, torch.full_like(target, -100), reduction=reduction)
    assert torch.isnan(loss) if reduction == "mean" else (loss == 0).all()
    for d in torch.autograd.grad(loss, (h, w), torch.ones_like(loss)):
        assert (d == 0).all()


@pytest.mark.parametrize("up", [1e-25, 1e-6, 1e6, 1e25])
def test_few_float_rows_of_any_scale(up):
    hidden, weight, target = make(40, 100, 600, torch.float32)
    check(hidden * up, weight / up, target)
    hidden[::2] *= 2.0 ** -20
    check(hidden, weight, target, "none")


@pytest.mark.parametrize("dtype", DTYPES)
def test_few_rows_with_large_logits(dtype):
    hidden, weight, target = make(40, 64, 600, dtype, scale=400.0)
    h, w = hidden.requires_grad_(), weight.requires_grad_()
    loss = tb.linear_cross_entropy(h, w, target)
    want, want_h, want_w = reference(h, w, target, torch.ones((), device="cuda"), "mean")
    assert abs(float(loss) - float(want)) < 1e-5 * (1 + abs(float(want)))
    dh, dw = torch.autograd.grad(loss, (h, w))
    assert err(dh, want_h) < max(2e-3, TOL[dtype]) and err(dw, want_w) < max(2e-3, TOL[dtype])


def test_few_rows_gradients_of_one_operand_alone_and_zero_upstream():
    hidden, weight, target = make(50, 64, 500, torch.float32)
    h, w = hidden.requires_grad_(), weight.requires_grad_()
    both = torch.autograd.grad(tb.linear_cross_entropy(h, w, target), (h, w))
    assert torch.equal(torch.autograd.grad(tb.linear_cross_entropy(h, w.detach(), target), h)[0], both[0])
    assert torch.equal(torch.autograd.grad(tb.linear_cross_entropy(h.detach(), w, target), w)[0], both[1])
    for reduction in ("mean", "none"):
        loss = tb.linear_cross_entropy(h, w, target, reduction=reduction)
        for d in torch.autograd.grad(loss, (h, w), torch.zeros_like(loss)):
            assert (d == 0).all()
    g = torch.logspace(-6, 2, 50, device="cuda")
    each = tb.linear_cross_entropy(h, w, target, reduction="none")
    dh, dw = torch.autograd.grad(each, (h, w), g)
    _, want_h, want_w = reference(h, w, target, g, "none")
    assert err(dh, want_h) < 5e-5 and err(dw, want_w) < 5e-5


@pytest.mark.parametrize("dtype", DTYPES)
def test_few_rows_same_bits_every_time_and_in_a_graph(dtype):
    hidden, weight, target = make(48, 200, 40000, dtype)
    first = check(hidden, weight, target)
    for a, b in zip(first, check(hidden, weight, target)):
        assert torch.equal(a, b)
    w = weight.detach().requires_grad_()
    grad = torch.ones((), device="cuda")
    step = tb.GraphedStep(lambda h: tb.linear_cross_entropy(h, w, target), hidden, grad, params=(w,))
    for k in range(3):
        h = (hidden * (1 + k)).requires_grad_()
        loss, grads = step(h.detach(), grad)
        torch.cuda.synchronize()
        want = tb.linear_cross_entropy(h, w, target)
        assert torch.equal(loss, want)
        for a, b in zip(grads, torch.autograd.grad(want, (h, w), grad)):
            assert torch.equal(a, b)


def test_refusals():
    hidden, weight, target = make(8, 16, 50, torch.float32)
    for call in (
        lambda: tb.linear_cross_entropy(hidden, weight[:, :8], target), lambda: tb.linear_cross_entropy(hidden, weight, target[:7]),
        lambda: tb.linear_cross_entropy(hidden, weight, target.int()), lambda: tb.linear_cross_entropy(hidden.half(), weight.half(), target),
        lambda: tb.linear_cross_entropy(hidden.bfloat16(), weight, target), lambda: tb.linear_cross_entropy(hidden, weight, target.cpu()),
        lambda: tb.linear_cross_entropy(hidden, weight[:0], target), lambda: tb.linear_cross_entropy(hidden, weight, target, reduction="all"),
        lambda: torch.ops.torch_butterfly.linear_cross_entropy(hidden.cpu(), weight.cpu(), target.cpu(), -100, 1),
        lambda: torch.ops.torch_butterfly.linear_cross_entropy(hidden, weight, target, -100, 3),
    ):
        with pytest.raises((RuntimeError, ValueError)):
            call()
