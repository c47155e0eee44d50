"""The gated linear recurrence against its definition in 64 bits, step by step on the host.

Errors are max |error| / max |reference|.  float32 and complex64: decays below one forget, so a value
carries the rounding of the last 1 / (1 - a) steps, each some four roundings of 2^-24, and what the runs of a
tile are composed from as many again: 1e-5.  bfloat16: results are rounded once (2^-9), and the gates' gradients
take the rounded h (2^-9 again, of h where h - x is asked for): 2^-6 of the largest."""
import pytest
import torch

import butterfly_amd as tb

pytestmark = pytest.mark.gpu

KINDS = [(torch.float32, True), (torch.float32, False), (torch.bfloat16, True), (torch.bfloat16, False), (torch.complex64, False)]
TOL = {torch.float32: 1e-5, torch.complex64: 1e-5, torch.bfloat16: 2.0 ** -6}


def wide_type(dtype):
    return torch.complex128 if dtype.is_complex else torch.float64


def state_type(dtype):
    return torch.float32 if dtype == torch.bfloat16 else dtype


def make(batch, steps, channels, dtype, sigmoid, seed=0):
    gen = torch.Generator().manual_seed(seed + 1000 * batch + 10 * steps + channels)

    def randn(*shape, dtype=dtype):
        return torch.randn(*shape, generator=gen, dtype=torch.complex64 if dtype.is_complex else torch.float32).to(dtype)

    gate = randn(batch, steps, channels) + 1
    if not sigmoid:
        turn = torch.exp(2j * gate.imag) if dtype.is_complex else 1.0
        gate = (torch.sigmoid(gate.real.float()) * turn).to(dtype)
    st = state_type(dtype)
    return {"gate": gate, "x": randn(batch, steps, channels), "state": randn(batch, channels, dtype=st),
            "grad": randn(batch, steps, channels), "grad_last": randn(batch, channels, dtype=st)}


def reference(v, sigmoid, reset=None, with_state=True):
    gate, x, g, gl = (v[k].cpu().to(wide_type(v["x"].dtype)) for k in ("gate", "x", "grad", "grad_last"))
    batch, steps, channels = x.shape
    h = v["state"].cpu().to(x.dtype) if with_state else torch.zeros(batch, channels, dtype=x.dtype)
    a = torch.sigmoid(gate) if sigmoid else gate
    rest = torch.sigmoid(-gate) if sigmoid else torch.ones_like(gate)
    hs, before = [], []
    zero = torch.zeros((), dtype=x.dtype)
    for t in range(steps):
        p = h if reset is None else torch.where(reset.cpu()[:, t, None], zero, h)
        before.append(p)
        h = (a[:, t] * p if reset is None else torch.where(reset.cpu()[:, t, None], zero, a[:, t] * p)) + rest[:, t] * x[:, t]
        hs.append(h)
    out = {"h": torch.stack(hs, 1), "last": h}
    d_gate, d_x, c = torch.empty_like(x), torch.empty_like(x), gl
    for t in reversed(range(steps)):
        e = g[:, t] + c
        d_gate[:, t] = e * (before[t] - x[:, t]) * a[:, t] * rest[:, t] if sigmoid else e * before[t].conj()
        d_x[:, t] = e * rest[:, t]
        c = a[:, t].conj() * e
        if reset is not None:
            c = torch.where(reset.cpu()[:, t, None], zero, c)
    out.update(d_gate=d_gate, d_x=d_x, d_state=c)
    return out


def close(got, want, tol, what):
    got, want = got.detach().cpu().to(want.dtype), want
    assert got.shape == want.shape
    if want.numel():
        e = float((got - want).abs().max() / want.abs().max().clamp(min=1e-30))
        assert e < tol, (what, e)


def check(v, sigmoid, reset=None, with_state=True):
    dtype = v["x"].dtype
    ref = reference(v, sigmoid, reset, with_state)
    d = {k: t.cuda() for k, t in v.items()}
    gate, x = d["gate"].requires_grad_(), d["x"].requires_grad_()
    state = d["state"].requires_grad_() if with_state else None
    h, last = tb.gated_recurrence(gate, x, state, None if reset is None else reset.cuda(), sigmoid)
    assert h.dtype == dtype and last.dtype == state_type(dtype)
    wanted = [gate, x] + ([state] if with_state else [])
    grads = torch.autograd.grad((h, last), wanted, (d["grad"], d["grad_last"]))
    close(h, ref["h"], TOL[dtype], "h")
    close(last, ref["last"], 1e-5, "last")
    for got, name in zip(grads, ("d_gate", "d_x", "d_state")):
        close(got, ref[name], 1e-5 if name == "d_state" else TOL[dtype], name)
    return h, last, grads


@pytest.mark.parametrize("dtype,sigmoid", KINDS)
@pytest.mark.parametrize("steps", [1, 2, 7, 8, 9, 31, 63, 64, 65, 127, 128, 129, 300])
def test_lengths(steps, dtype, sigmoid):
    check(make(2, steps, 70, dtype, sigmoid), sigmoid)


@pytest.mark.parametrize("dtype,sigmoid", KINDS)
@pytest.mark.parametrize("channels", [1, 2, 3, 63, 64, 65, 127, 128, 129, 257])
def test_channels(channels, dtype, sigmoid):
    check(make(3, 40, channels, dtype, sigmoid), sigmoid, with_state=channels % 2 == 0)


@pytest.mark.parametrize("dtype,sigmoid", KINDS)
@pytest.mark.parametrize("batch,steps,channels", [(1, 2050, 64), (1, 1500, 3), (2, 1000, 200), (5, 777, 31)])
def test_few_channels_and_many_steps_are_cut_into_chunks(batch, steps, channels, dtype, sigmoid):
    v = make(batch, steps, channels, dtype, sigmoid)
    check(v, sigmoid)
    gen = torch.Generator().manual_seed(steps)
    check(v, sigmoid, torch.rand(batch, steps, generator=gen) < 0.01, with_state=False)


@pytest.mark.parametrize("dtype,sigmoid", KINDS)
def test_many_sequences_stay_whole(dtype, sigmoid):
    check(make(200, 150, 65, dtype, sigmoid), sigmoid)


@pytest.mark.parametrize("dtype,sigmoid", KINDS)
@pytest.mark.parametrize("share", [0.02, 0.5, 1.0])
def test_resets(share, dtype, sigmoid):
    v = make(3, 300, 66, dtype, sigmoid)
    gen = torch.Generator().manual_seed(3)
    reset = torch.rand(3, 300, generator=gen) < share
    check(v, sigmoid, reset)
    reset[:] = False
    reset[0, 0] = reset[1, 299] = True
    check(v, sigmoid, reset)
    # other strides of the marks
    check(v, sigmoid, reset.t().contiguous().t())
    check(v, sigmoid, reset[:1].expand(3, 300))


@pytest.mark.parametrize("dtype,sigmoid", KINDS)
@pytest.mark.parametrize("share", [0.5, 1.0])
def test_resets_in_chunks(share, dtype, sigmoid):
    v = make(2, 1111, 66, dtype, sigmoid)
    reset = torch.rand(2, 1111, generator=torch.Generator().manual_seed(4)) < share
    check(v, sigmoid, reset)
    reset[:] = False
    reset[0, 0] = reset[1, 1110] = True
    check(v, sigmoid, reset)


@pytest.mark.parametrize("steps,where", [(40, 13), (300, 200), (1200, 700)])
@pytest.mark.parametrize("dtype,sigmoid", KINDS)
def test_nothing_from_before_a_reset_gets_through(steps, where, dtype, sigmoid):
    v = make(1, steps, 30, dtype, sigmoid)
    reset = torch.zeros(1, steps, dtype=torch.bool)
    reset[0, where] = True
    clean = {k: t.cuda() for k, t in v.items()}
    marks = reset.cuda()
    h0, last0 = tb.gated_recurrence(clean["gate"], clean["x"], clean["state"], marks, sigmoid)
    for bad in (float("inf"), float("nan")):
        x = clean["x"].clone()
        x[0, where // 2] = bad
        state = clean["state"].clone()
        state[0, 3] = bad
        x.requires_grad_()
        h, last = tb.gated_recurrence(clean["gate"], x, state, marks, sigmoid)
        assert torch.equal(h[:, where:], h0[:, where:]) and torch.equal(last, last0)
        assert not torch.isfinite(torch.view_as_real(h) if h.is_complex() else h)[0, where - 1].all()
        # nor does a gradient from behind it
        grad = torch.zeros_like(h)
        grad[0, where + 1] = bad
        dx, = torch.autograd.grad(h, x, grad)
        dx = torch.view_as_real(dx) if dx.is_complex() else dx
        assert (dx[0, :where // 2] == 0).all() and (dx[0, where // 2 + 1:where] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gates_at_their_ends(dtype):
    v = make(2, 50, 40, dtype, True)
    v["gate"][:, ::3] = 100.0
    v["gate"][:, 1::3] = -100.0
    check(v, True)
    v["gate"][:, ::3] = float("inf")
    v["gate"][:, 1::3] = float("-inf")
    check(v, True)
    # close to one the rest is not lost to a difference
    v["gate"][:] = 12.0
    check(v, True)


@pytest.mark.parametrize("dtype,sigmoid", KINDS)
def test_strides(dtype, sigmoid):
    v = make(4, 90, 50, dtype, sigmoid)
    ref = reference(v, sigmoid)
    packed = torch.cat((v["gate"], v["x"]), -1).cuda()
    seconds = packed.transpose(0, 1).contiguous().transpose(0, 1)      # steps outside, batch inside
    columns = packed.transpose(1, 2).contiguous().transpose(1, 2)      # channels not adjacent
    for p in (packed, seconds, columns):
        leaf = p.detach().requires_grad_()
        gate, x = leaf.chunk(2, -1)
        h, last = tb.gated_recurrence(gate, x, v["state"].cuda(), None, sigmoid)
        close(h, ref["h"], TOL[dtype], "h")
        for g in (v["grad"].cuda(), v["grad"].cuda().transpose(1, 2).contiguous().transpose(1, 2)):
            d, = torch.autograd.grad((h, last), leaf, (g, v["grad_last"].cuda()), retain_graph=True)
            close(d, torch.cat((ref["d_gate"], ref["d_x"]), -1), TOL[dtype], "d")


def test_one_of_the_two_gradients_alone_and_broadcast_ones():
    v = make(2, 33, 20, torch.float32, True)
    d = {k: t.cuda() for k, t in v.items()}
    gate, x = d["gate"].requires_grad_(), d["x"].requires_grad_()
    h, last = tb.gated_recurrence(gate, x)
    zero = torch.zeros_like
    for outs, grads, gv in (((h,), (d["grad"],), {"grad_last": zero(v["grad_last"])}),
                            ((last,), (d["grad_last"],), {"grad": zero(v["grad"])})):
        ref = reference({**v, **gv}, True, with_state=False)
        got = torch.autograd.grad(outs, (gate, x), grads, retain_graph=True)
        close(got[0], ref["d_gate"], 1e-5, "d_gate")
        close(got[1], ref["d_x"], 1e-5, "d_x")
    got = torch.autograd.grad(h.sum(), (gate, x))
    ref = reference({**v, "grad": torch.ones_like(v["grad"]), "grad_last": zero(v["grad_last"])}, True, with_state=False)
    close(got[0], ref["d_gate"], 1e-5, "d_gate")
    # one row of gates and inputs for all sequences
    one = v["gate"][:1].cuda().requires_grad_()
    h, _ = tb.gated_recurrence(one.expand(2, 33, 20), x)
    d_one, = torch.autograd.grad(h, one, d["grad"])
    ref = reference({**v, "gate": v["gate"][:1].expand(2, 33, 20), "grad_last": zero(v["grad_last"])}, True, with_state=False)
    close(d_one, ref["d_gate"].sum(0, keepdim=True), 1e-5, "d_gate")


def test_no_steps_and_no_sequences():
    for batch, steps, channels in ((2, 0, 5), (0, 4, 5), (2, 4, 0)):
        gate = torch.zeros(batch, steps, channels, device="cuda", requires_grad=True)
        state = torch.randn(batch, channels, device="cuda").requires_grad_()
        h, last = tb.gated_recurrence(gate, gate.detach(), state)
        assert h.shape == (batch, steps, channels)
        if steps == 0:
            assert torch.equal(last, state)
            g = torch.randn_like(state)
            ds, = torch.autograd.grad(last, state, g)
            assert torch.equal(ds, g)
            assert torch.equal(tb.gated_recurrence(gate, gate)[1], torch.zeros_like(state))


@pytest.mark.parametrize("dtype,sigmoid", KINDS)
@pytest.mark.parametrize("channels", [1, 33, 128, 600])
def test_token_by_token_equals_the_sequence(channels, dtype, sigmoid):
    v = {k: t.cuda() for k, t in make(3, 20, channels, dtype, sigmoid).items()}
    ref = reference(v, sigmoid)
    state = v["state"].clone()
    version = state._version
    for t in range(20):
        h = tb.gated_recurrence_step(v["gate"][:, t], v["x"][:, t], state, sigmoid)
        close(h, ref["h"][:, t], TOL[dtype], t)
    close(state, ref["last"], 1e-5, "state")
    assert state._version > version


def test_gradients_against_differences():
    """Along random directions with a step of 1/64: the third derivative's share and the rounding of the values both
    stay below 2e-3 of the derivative's scale."""
    v = {k: t.cuda() for k, t in make(2, 60, 10, torch.float32, True).items()}
    reset = torch.zeros(2, 60, dtype=torch.bool, device="cuda")
    reset[0, 20] = True

    def value(gate, x, state):
        h, last = tb.gated_recurrence(gate, x, state, reset)
        return float((h.double() * v["grad"]).sum() + (last.double() * v["grad_last"]).sum())

    args = [v["gate"], v["x"], v["state"]]
    leaves = [a.clone().requires_grad_() for a in args]
    grads = torch.autograd.grad(tb.gated_recurrence(*leaves, reset), leaves, (v["grad"], v["grad_last"]))
    for k, grad in enumerate(grads):
        d = torch.randn(args[k].shape, generator=torch.Generator().manual_seed(k)).cuda()
        up, down = list(args), list(args)
        up[k], down[k] = args[k] + d / 64, args[k] - d / 64
        numeric = (value(*up) - value(*down)) * 32
        assert abs(numeric - float((grad.double() * d).sum())) < 2e-3 * float(grad.double().norm() * d.double().norm()), k


@pytest.mark.parametrize("shape", [(16, 600, 256), (1, 3000, 100)])
def test_same_bits_every_time_and_on_another_stream(shape):
    v = make(*shape, torch.float32, True)
    first = check(v, True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = check(v, True)
    for a, b in zip((*first[:2], *first[2]), (*again[:2], *again[2])):
        assert torch.equal(a, b)


def test_in_a_graph():
    v = {k: t.cuda() for k, t in make(1, 1000, 60, torch.float32, True).items()}
    step = tb.GraphedStep(lambda x: tb.gated_recurrence(v["gate"], x, v["state"])[0], v["x"], v["grad"])
    for k in range(3):
        x = v["x"] * (k + 1)
        y, (dx,) = step(x, v["grad"])
        torch.cuda.synchronize()
        leaf = x.clone().requires_grad_()
        h, _ = tb.gated_recurrence(v["gate"], leaf, v["state"])
        assert torch.equal(y, h) and torch.equal(dx, torch.autograd.grad(h, leaf, v["grad"])[0])


def test_refusals():
    x = torch.zeros(2, 5, 8, device="cuda")
    c = x.to(torch.complex64)
    for call in (
        lambda: tb.gated_recurrence(x[:, :4], x), lambda: tb.gated_recurrence(x.bfloat16(), x), lambda: tb.gated_recurrence(x[0], x[0]),
        lambda: tb.gated_recurrence(c, c), lambda: tb.gated_recurrence(x.half(), x.half()), lambda: tb.gated_recurrence(x.cpu(), x),
        lambda: tb.gated_recurrence(x, x, torch.zeros(2, 7, device="cuda")), lambda: tb.gated_recurrence(x, x, x[:, 0].bfloat16()),
        lambda: tb.gated_recurrence(x, x, None, torch.zeros(2, 5, device="cuda")),
        lambda: tb.gated_recurrence(x, x, None, torch.zeros(2, 4, dtype=torch.bool, device="cuda")),
        lambda: tb.gated_recurrence_step(x, x, x[:, 0]), lambda: tb.gated_recurrence_step(x[:, 0], x[:, 0], torch.zeros(8, 2, device="cuda").t()),
        lambda: tb.gated_recurrence_step(x[:, 0].clone().requires_grad_(), x[:, 0], torch.zeros(2, 8, device="cuda")),
        lambda: torch.ops.torch_butterfly.gated_recurrence(x.cpu(), x.cpu(), None, None, True),
    ):
        with pytest.raises(RuntimeError):
            call()
    gate = x.clone().requires_grad_()
    h, _ = tb.gated_recurrence(gate, x)
    with torch.no_grad():
        h.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(h.sum(), gate)
