"""The loss at the edges of what it is given: what lies behind and between the weight's rows, rows and gradients that are not
finite or of unlike size, empty batches.  Error measure and tolerances are those of the loss's other tests."""
import pytest
import torch

import butterfly_amd as tb
from test_gpu_linear_cross_entropy import DTYPES, TOL, check, err, make, reference

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,features,vocab", [(70, 64, 1000), (300, 72, 1000), (300, 64, 100), (2048, 64, 16390), (3000, 1024, 4100)])
def test_what_lies_behind_the_weight_reaches_nothing(rows, features, vocab, dtype):
    """The last k step of the hidden rows' gradient and the last tile of the logits end inside a step and a tile: NaN behind
    the weight's last row would show in either."""
    hidden, weight, target = make(rows, features, vocab, dtype)
    tall = torch.full((vocab + 300, features), float("nan"), dtype=dtype, device="cuda")
    tall[:vocab] = weight
    for a, b in zip(check(hidden, tall[:vocab], target), check(hidden, weight, target)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
def test_no_rows_give_the_weight_no_gradient(reduction, dtype):
    hidden, weight, target = make(0, 40, 777, dtype)
    # (memory that the operators take next is not zero)
    used = [torch.full((1 << k,), float("nan"), device="cuda") for k in range(8, 22)]
    del used
    h, w = hidden.requires_grad_(), weight.requires_grad_()
    loss = tb.linear_cross_entropy(h, w, target, reduction=reduction)
    dh, dw = torch.autograd.grad(loss, (h, w), torch.ones_like(loss))
    assert dh.shape == (0, 40) and torch.equal(dw, torch.zeros_like(weight))


@pytest.mark.parametrize("gap", [8, 24, 64])
@pytest.mark.parametrize("rows,features,vocab", [(70, 40, 1000), (300, 200, 515), (2048, 72, 16390), (3000, 1000, 4100)])
def test_what_lies_between_the_weights_rows_reaches_nothing(rows, features, vocab, gap):
    """bfloat16 rows that 16 bytes divide are read where they lie, by steps of 64 features that end inside the gap."""
    hidden, weight, target = make(rows, features, vocab, torch.bfloat16)
    wide = torch.full((vocab, features + gap), float("nan"), dtype=torch.bfloat16, device="cuda")
    wide[:, :features] = weight
    for a, b in zip(check(hidden, wide[:, :features], target), check(hidden, weight, target)):
        assert torch.equal(a, b)


def test_an_entry_of_no_probability_spoils_no_other_entry():
    """Weight rows with an entry of minus infinity give a logit of minus infinity (positive hidden features): nothing of
    them may reach the entry in front, whose last k step ends where they begin."""
    hidden, weight, target = make(80, 72, 500, torch.bfloat16)
    hidden = hidden.abs() + 0.125
    target = target.masked_fill(target == 7, 8)
    weight[7, 3] = float("-inf")
    loss = tb.linear_cross_entropy(hidden, weight, target, reduction="none")
    logits = hidden.double() @ weight.double().t()
    want = torch.nn.functional.cross_entropy(logits, target, reduction="none")
    assert (loss.double() - want).abs().max() < 1e-5 * (1 + want.abs().max())


@pytest.mark.parametrize("up", [1e-6, 1e-3, 1.0, 1e5])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [40, 90, 700])
def test_a_row_that_is_not_finite_spoils_no_other(rows, dtype, up):
    """Losses and hidden gradients of the other rows; every row of the weight's gradient sums over all of them."""
    hidden, weight, target = make(rows, 64, 1000, dtype, ignored=0.0)
    hidden, weight = hidden * up, weight / up
    good = torch.ones(rows, dtype=torch.bool, device="cuda")
    good[[3, 11, rows - 1]] = False
    h, w = hidden.clone(), weight.requires_grad_()
    h[3, 5], h[11, 0], h[rows - 1, 63] = float("nan"), float("inf"), float("-inf")
    h.requires_grad_()
    each = tb.linear_cross_entropy(h, w, target, reduction="none")
    dh, dw = torch.autograd.grad(each, (h, w), torch.ones_like(each))
    want, want_h, _ = reference(hidden[good], weight, target[good], torch.ones(int(good.sum()), device="cuda"), "none")
    assert (each[good].double() - want).abs().max() <= 1e-5 * (1 + want.abs().max())
    assert err(dh[good], want_h) < TOL[dtype]
    assert not torch.isfinite(each[~good]).any() and not torch.isfinite(dh[~good]).any() and not torch.isfinite(dw).any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [40, 90, 700])
def test_a_rows_gradient_that_is_not_finite_spoils_no_other_row(rows, dtype):
    hidden, weight, target = make(rows, 64, 1000, dtype, ignored=0.0)
    good = torch.ones(rows, dtype=torch.bool, device="cuda")
    good[[3, 11, rows - 1]] = False
    g = torch.linspace(0.5, 2.0, rows, device="cuda")
    _, want_h, _ = reference(hidden, weight, target, g, "none")
    g[3], g[11], g[rows - 1] = float("nan"), float("inf"), float("-inf")
    h, w = hidden.requires_grad_(), weight.requires_grad_()
    dh, dw = torch.autograd.grad(tb.linear_cross_entropy(h, w, target, reduction="none"), (h, w), g)
    assert err(dh[good], want_h[good]) < TOL[dtype]
    assert not torch.isfinite(dh[~good]).any() and not torch.isfinite(dw).any()
    # nothing but zeros beside it
    g[good] = 0.0
    dh, = torch.autograd.grad(tb.linear_cross_entropy(h, w, target, reduction="none"), h, g)
    assert (dh[good] == 0).all() and not torch.isfinite(dh[~good]).any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", [(50, 1000), (300, 1000), (700, 9000)])
def test_every_row_keeps_its_bits_whatever_the_others_gradients(rows, vocab, dtype):
    """A row of d_hidden is g (sum_v p_v W_v - W_t): off by the tolerance times g and the largest weight, its own g, be it
    10^-30 of the largest."""
    hidden, weight, target = make(rows, 64, vocab, dtype)
    h, w = hidden.requires_grad_(), weight.requires_grad_()
    g = torch.logspace(-30, 0, rows, device="cuda")[torch.randperm(rows, generator=torch.Generator().manual_seed(1)).cuda()]
    g[5] = 0.0
    dh, dw = torch.autograd.grad(tb.linear_cross_entropy(h, w, target, reduction="none"), (h, w), g)
    _, want_h, want_w = reference(h, w, target, g, "none")
    off = (dh.double() - want_h).abs().amax(1) / (g.double() * float(w.detach().abs().max())).clamp(min=1e-300)
    assert off.max() < TOL[dtype] and (dh[5] == 0).all() and err(dw, want_w) < TOL[dtype]


@pytest.mark.parametrize("rows", [40, 90, 700])
def test_float_operands_far_apart(rows):
    """Hidden rows of some 2^112 and weights of some 2^-100: logits of some 2^15, off by 2^-20 of that (1e-5 of the losses)."""
    hidden, weight, target = make(rows, 64, 1000, torch.float32, ignored=0.0)
    hidden, weight = hidden * 2.0 ** 112, weight * 2.0 ** -100
    each = tb.linear_cross_entropy(hidden, weight, target, reduction="none")
    want, _, _ = reference(hidden, weight, target, torch.ones(rows, device="cuda"), "none")
    assert (each.double() - want).abs().max() <= 1e-5 * (1 + want.abs().max())


def test_a_weight_whose_features_are_not_adjacent_is_copied_once():
    hidden, weight, target = make(70, 256, 20000, torch.bfloat16)
    columns = weight.t().contiguous().t().requires_grad_()
    tb.linear_cross_entropy(hidden, columns, target)
    before = torch.cuda.memory_stats()["allocated_bytes.all.allocated"]
    tb.linear_cross_entropy(hidden, columns, target)
    assert torch.cuda.memory_stats()["allocated_bytes.all.allocated"] - before < 1.5 * weight.numel() * 2


@pytest.mark.parametrize("up", [1e5, 1e7, 1e10, 1e15])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [40, 90, 700])
def test_logits_of_any_size(rows, dtype, up):
    """A softmax of far larger logits is one-hot but for ties: losses off by 2^-20 of the logits (1e-5 of the largest loss), and
    gradients of at most two rows' sum."""
    hidden, weight, target = make(rows, 64, 1000, dtype, ignored=0.0)
    h, w = (hidden * up).requires_grad_(), (weight * up).requires_grad_()
    each = tb.linear_cross_entropy(h, w, target, reduction="none")
    want, _, _ = reference(h, w, target, torch.ones(rows, device="cuda"), "none")
    assert (each.double() - want).abs().max() <= 1e-5 * (1 + want.abs().max())
    dh, dw = torch.autograd.grad(each, (h, w), torch.ones_like(each))
    assert torch.isfinite(dh).all() and float(dh.abs().max()) <= 2.1 * float(w.abs().max())
    assert torch.isfinite(dw).all() and float(dw.abs().max()) <= 1.1 * rows * float(h.abs().max())


@pytest.mark.parametrize("rows", [50, 100, 1000])
def test_unlikely_entries_keep_their_bits(rows):
    """Every entry of the weight's gradient by itself: sums of the entry's probabilities, all of one size.  float32: 2^-20 of a
    logit of up to 28, and pairs of 22 bits for probabilities from 2^-28 up, of 11 down to 2^-40."""
    gen = torch.Generator().manual_seed(rows)
    logits = -torch.linspace(0, 40, 401, dtype=torch.float64) * torch.log(torch.tensor(2.0, dtype=torch.float64))
    h, w = torch.zeros(rows, 64), torch.zeros(401, 64)
    h[:, 0], w[:, 0] = 1.0, logits.float()
    h[:, 1:] = torch.rand(rows, 63, generator=gen)      # (against weights of zero)
    h, w = h.cuda().requires_grad_(), w.cuda().requires_grad_()
    target = torch.zeros(rows, dtype=torch.int64, device="cuda")
    dw, = torch.autograd.grad(tb.linear_cross_entropy(h, w, target, reduction="sum"), w)
    _, _, want = reference(h, w, target, torch.ones((), device="cuda"), "sum")
    off = ((dw.double() - want).abs() / want.abs()).amax(1).cpu()
    p = torch.softmax(w.detach()[:, 0].double(), 0).cpu()
    assert off[p >= 2.0 ** -28].max() < 5e-5
    assert off[p >= 2.0 ** -40].max() < 2.0 ** -11


@pytest.mark.parametrize("rows", [50, 100, 700])
def test_float_rows_and_features_of_unlike_scale(rows):
    """Numbers from 2^-28 of the operand's largest up keep 22 bits, and a few below that 20."""
    hidden, weight, target = make(rows, 64, 1000, torch.float32, ignored=0.0)
    ones = torch.ones(rows, device="cuda")
    # features: every product as it was
    scale = torch.full((64,), 2.0 ** 13, device="cuda")
    scale[::2] = 2.0 ** -13
    h, w = (hidden * scale).requires_grad_(), (weight / scale).requires_grad_()
    each = tb.linear_cross_entropy(h, w, target, reduction="none")
    want, want_h, want_w = reference(h, w, target, ones, "none")
    assert (each.double() - want).abs().max() <= 1e-5 * (1 + want.abs().max())
    dh, dw = torch.autograd.grad(each, (h, w), ones)
    for part in (slice(0, None, 2), slice(1, None, 2)):
        assert err(dh[:, part], want_h[:, part]) < TOL[torch.float32] and err(dw[:, part], want_w[:, part]) < TOL[torch.float32]
    # rows: ordinary logits beside enormous ones
    h, w = hidden * 2.0 ** 13, (weight * 2.0 ** 13).requires_grad_()
    h[::2] = hidden[::2] * 2.0 ** -13
    h.requires_grad_()
    each = tb.linear_cross_entropy(h, w, target, reduction="none")
    want, want_h, _ = reference(h, w, target, ones, "none")
    assert (each[::2].double() - want[::2]).abs().max() <= 1e-5 * (1 + want[::2].abs().max())
    dh, = torch.autograd.grad(each, h, ones)
    assert err(dh[::2], want_h[::2]) < TOL[torch.float32]
