"""Rotary positions against the formula in 64 bits.

float32: an angle, reduced to a turn, is off by 2^-25 of a turn (2 pi 2^-25 < 2^-22) and its cosine by some 2^-23, products and sums by
2^-23 more: 2^-20 of the largest feature.  bfloat16: results are rounded once, 2^-8."""
import pytest
import torch

import butterfly_amd as tb

pytestmark = pytest.mark.gpu


def reference(x, positions, frequencies, interleaved, magnitude, sign=1.0):
    pairs = frequencies.shape[0]
    x = x.detach().cpu().double()
    angle = sign * positions.cpu().double()[..., None, None] * frequencies.cpu()
    z = torch.polar(torch.full((), magnitude, dtype=torch.float64), angle)
    one = torch.arange(pairs) * (2 if interleaved else 1)
    two = one + (1 if interleaved else pairs)
    y = x.clone()
    turned = torch.complex(x[..., one], x[..., two]) * z
    y[..., one], y[..., two] = turned.real, turned.imag
    return y


def tolerance(dtype):
    return 2.0 ** -20 if dtype == torch.float32 else 2.0 ** -8 + 2.0 ** -20


def check(got, want, dtype, magnitude=1.0):
    assert got.dtype == dtype and got.shape == want.shape
    if want.numel():
        assert float((got.detach().double().cpu() - want).abs().max() / want.abs().max()) <= tolerance(dtype)


SHAPES = [((1, 1), 1, 2, 2), ((2, 3), 2, 16, 16), ((5,), 4, 64, 64), ((2, 37), 3, 100, 50), ((1, 129), 1, 6, 4), ((3, 7), 5, 34, 34), ((), 3, 18, 10),
          ((2, 3, 4), 2, 24, 24), ((1, 3), 2, 20, 0), ((2, 300), 16, 64, 64), ((1, 2), 1, 4096, 4096), ((7,), 33, 128, 2)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
def test_against_the_formula(shape, interleaved, dtype):
    lead, heads, features, rotated = shape
    gen = torch.Generator().manual_seed(features + rotated)
    x, g = (torch.randn(*lead, heads, features, generator=gen).to(dtype) for _ in range(2))
    positions = torch.randint(0, 5000, lead, generator=gen)
    frequencies = tb.rotary_frequencies(rotated)[0] if rotated else torch.zeros(0, dtype=torch.float64)
    leaf = x.cuda().requires_grad_()
    y = tb.rotary(leaf, positions.cuda(), frequencies.cuda(), interleaved, 1.5)
    check(y, reference(x, positions, frequencies, interleaved, 1.5), dtype)
    d, = torch.autograd.grad(y, leaf, g.cuda())
    check(d, reference(g, positions, frequencies, interleaved, 1.5, -1.0), dtype)
    if rotated < features:
        assert torch.equal(y[..., rotated:], leaf[..., rotated:]) and torch.equal(d[..., rotated:].cpu(), g[..., rotated:])


@pytest.mark.parametrize("position", [0, 1, -7, 65536, 10 ** 6 + 1, 2 ** 31 + 5, -(2 ** 31) - 3])
def test_far_positions(position):
    # off by the rounding of a turn's fraction in 64 bits, 2^31 / (2 pi) 2^-52: below the rest
    frequencies = tb.rotary_frequencies(64)[0]
    x = torch.randn(3, 2, 64)
    positions = torch.full((3,), position)
    check(tb.rotary(x.cuda(), positions.cuda(), frequencies.cuda()), reference(x, positions, frequencies, False, 1.0), torch.float32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_second_derivatives(dtype):
    frequencies = tb.rotary_frequencies(20)[0].cuda()
    fused = torch.randn(3, 40, 6, 24, device="cuda").to(dtype)
    positions = torch.arange(40, device="cuda").expand(3, 40)
    want = reference(fused, positions, frequencies, False, 1.0)
    check(tb.rotary(fused[:, :, 2:5], positions, frequencies), want[:, :, 2:5], dtype)
    check(tb.rotary(fused.transpose(0, 1), positions.t(), frequencies), want.transpose(0, 1), dtype)
    check(tb.rotary(fused[::2, 1::3], positions[::2, 1::3], frequencies), want[::2, 1::3], dtype)
    check(tb.rotary(fused.permute(0, 1, 3, 2).contiguous().permute(0, 1, 3, 2), positions, frequencies), want, dtype)
    check(tb.rotary(fused[:, :1].expand(3, 40, 6, 24), positions, frequencies), reference(fused[:, :1].expand(3, 40, 6, 24), positions, frequencies, False, 1.0), dtype)
    check(tb.rotary(fused[:, :, :, 1:23], positions, frequencies), reference(fused[:, :, :, 1:23], positions, frequencies, False, 1.0), dtype)
    x = fused.clone().requires_grad_()
    y = tb.rotary(x, positions, frequencies)
    g = torch.randn_like(y, requires_grad=True)
    d, = torch.autograd.grad(y, x, g, create_graph=True)
    check(d, reference(g, positions, frequencies, False, 1.0, -1.0), dtype)
    h = torch.randn_like(y)
    dd, = torch.autograd.grad(d, g, h)
    check(dd, reference(h, positions, frequencies, False, 1.0), dtype)


def test_nothing_to_do_and_refusals():
    frequencies = tb.rotary_frequencies(8)[0].cuda()
    for lead, heads in (((0, 4), 2), ((2, 0), 2), ((2, 3), 0)):
        x = torch.zeros(*lead, heads, 8, device="cuda", requires_grad=True)
        y = tb.rotary(x, torch.zeros(lead, dtype=torch.int64, device="cuda"), frequencies)
        assert y.shape == x.shape
        assert torch.autograd.grad(y.sum(), x)[0].shape == x.shape
    x, p = torch.zeros(2, 3, 2, 8, device="cuda"), torch.zeros(2, 3, dtype=torch.int64, device="cuda")
    for text, args in (("float32 and bfloat16", (x.double(), p, frequencies)), ("int64", (x, p.int(), frequencies)), ("shape of x", (x, p[:1], frequencies)),
                       ("float64", (x, p, frequencies.float())), ("more frequencies", (x[..., :6], p, frequencies)), ("on the device", (x, p.cpu(), frequencies)),
                       ("shape", (x[0, 0, 0], p, frequencies))):
        with pytest.raises(RuntimeError, match=text):
            tb.rotary(*args)


def test_captured_with_positions_that_move():
    frequencies = tb.rotary_frequencies(32)[0].cuda()
    x, positions = torch.randn(4, 2, 32, device="cuda"), torch.arange(4, device="cuda")
    graph = torch.cuda.CUDAGraph()
    tb.rotary(x, positions, frequencies)
    with torch.cuda.graph(graph):
        y = tb.rotary(x, positions, frequencies)
    for _ in range(3):
        positions += 1000
        graph.replay()
        torch.cuda.synchronize()
        check(y, reference(x, positions, frequencies, False, 1.0), torch.float32)


@pytest.mark.parametrize("lead", [(), (5,), (2, 3, 4), (0, 3)])
def test_any_number_of_dimensions_in_front(lead):
    gen = torch.Generator().manual_seed(1)
    x, positions = torch.randn(*lead, 3, 10, generator=gen), torch.randint(0, 1000, lead, generator=gen)
    frequencies, _ = tb.rotary_frequencies(8)
    got, want = tb.rotary(x.cuda(), positions.cuda(), frequencies.cuda()), tb.rotary(x.double(), positions, frequencies)
    assert got.shape == x.shape
    # (a sum of two products whose factors and whose sum are off by 2^-24 each, the angle by 2^-24 of a half turn)
    assert x.numel() == 0 or float((got.cpu() - want).abs().max()) <= 8 * 2.0 ** -24 * float(x.abs().max())
