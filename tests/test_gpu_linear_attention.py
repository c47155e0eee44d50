"""Linear attention with a decay for each head against its definition in 64 bits, step by step, gradients by automatic
differentiation of that.

Errors are max |error| / max |reference|.  float32: a result is a sum of some hundred products whose partial sums carry
2^-24 each, decays some four roundings each, over the chunks that a state remembers: 1e-5.  bfloat16: results are rounded once
(2^-8), what they are summed from has 16 bits: 2^-8 + 2^-12; with more than 64 features or values d_v also reads the
state's gradient in 8 bits, 2^-8 of each of its terms: 2^-7 + 2^-12.  States and their gradients are sums in 24
bits: 1e-5; the decays' gradients are sums of what has 16 bits: 2^-13."""
import pytest
import torch

import butterfly_amd as tb

pytestmark = pytest.mark.gpu

NAMES = ("q", "k", "v", "log_decay", "state")
HALF = 2.0 ** -8 + 2.0 ** -12


def tolerance(name, dtype, wide):
    if dtype == torch.float32 or name in ("last", "d_state"):
        return 1e-5
    if name == "d_log_decay":
        return 2.0 ** -13
    return HALF + (2.0 ** -8 if name == "d_v" and wide else 0.0)


def make(batch, steps, heads, groups, features, values, dtype, seed=0, slow=0.05):
    gen = torch.Generator().manual_seed(seed + 1000 * steps + 10 * features + values)

    def randn(*shape, dtype=dtype):
        return torch.randn(*shape, generator=gen).to(dtype)

    return {"q": randn(batch, steps, groups, features), "k": randn(batch, steps, groups, features), "v": randn(batch, steps, heads, values),
            "log_decay": -torch.rand(batch, steps, heads, generator=gen) * slow, "state": randn(batch, heads, features, values, dtype=torch.float32),
            "grad": randn(batch, steps, heads, values), "grad_last": randn(batch, heads, features, values, dtype=torch.float32)}


def reference(v, scale, reset=None, with_state=True, grads=("grad", "grad_last")):
    w = {k: t.detach().cpu().double() for k, t in v.items()}
    leaves = {k: w[k].requires_grad_() for k in NAMES}
    batch, steps, heads, _ = w["v"].shape
    shared = heads // w["q"].shape[2]
    q, k = (leaves[n].repeat_interleave(shared, 2) for n in "qk")
    s = leaves["state"] if with_state else torch.zeros_like(w["state"])
    out = []
    for t in range(steps):
        decayed = torch.exp(leaves["log_decay"][:, t])[..., None, None] * s
        if reset is not None:
            decayed = torch.where(reset.cpu()[:, t, None, None, None], torch.zeros(()).double(), decayed)
        s = decayed + k[:, t, :, :, None] * leaves["v"][:, t, :, None, :]
        out.append(scale * torch.einsum("bhd,bhde->bhe", q[:, t], s))
    o = torch.stack(out, 1)
    outs, gs = zip(*[(x, w[g]) for x, g in ((o, "grad"), (s, "grad_last")) if g in grads])
    wanted = NAMES if with_state else NAMES[:-1]
    d = torch.autograd.grad(outs, [leaves[n] for n in wanted], gs, allow_unused=True)
    result = {"o": o.detach(), "last": s.detach()}
    result.update(("d_" + n, g) for n, g in zip(wanted, d))
    return result


def device(v, scale, reset=None, with_state=True, grads=("grad", "grad_last")):
    leaves = {k: v[k].cuda().requires_grad_() for k in NAMES}
    o, last = tb.linear_attention(*(leaves[k] for k in NAMES[:4]), leaves["state"] if with_state else None,
                                  None if reset is None else reset.cuda(), scale)
    outs, gs = zip(*[(x, v[g].cuda()) for x, g in ((o, "grad"), (last, "grad_last")) if g in grads])
    wanted = NAMES if with_state else NAMES[:-1]
    d = torch.autograd.grad(outs, [leaves[n] for n in wanted], gs)
    result = {"o": o.detach(), "last": last.detach()}
    result.update(("d_" + n, g) for n, g in zip(wanted, d))
    return result


def compare(got, want, dtype, wide=False, scale=1.0):
    for name, w in want.items():
        g = got[name].double().cpu()
        assert g.shape == w.shape, name
        assert got[name].dtype == (torch.float32 if name in ("last", "d_state", "d_log_decay") else dtype), name
        err = float((g - w).abs().max() / w.abs().max().clamp(min=1e-30)) if w.numel() else 0.0
        assert err <= scale * tolerance(name, dtype, wide), (name, err)


SHAPES = [
    (1, 1, 1, 1, 1, 1), (2, 1, 3, 3, 64, 64), (1, 2, 1, 1, 16, 16), (2, 63, 2, 2, 64, 64), (1, 64, 2, 2, 32, 64), (3, 65, 2, 1, 64, 32),
    (1, 129, 3, 3, 17, 33), (2, 200, 4, 2, 64, 64), (1, 31, 2, 2, 128, 128), (2, 97, 2, 1, 128, 128), (1, 300, 6, 2, 100, 100),
    (1, 130, 1, 1, 65, 3), (1, 130, 1, 1, 3, 65), (1, 1000, 2, 2, 64, 64), (1, 700, 2, 1, 128, 72),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_against_the_definition(shape, dtype):
    v = make(*shape, dtype)
    scale = shape[4] ** -0.5
    compare(device(v, scale), reference(v, scale), dtype, wide=max(shape[4:]) > 64)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("heads", [200, 5])
def test_whole_sequences_and_segments(heads, dtype):
    # 200 heads fill the chip; five are cut into segments, some of them short
    v = make(1, 450, heads, heads, 20, 24, dtype)
    compare(device(v, 0.3), reference(v, 0.3), dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size", [64, 100])
def test_resets(size, dtype):
    v = make(3, 333, 2, 2, size, size, dtype)
    reset = torch.zeros(3, 333, dtype=torch.bool)
    reset[0, 0] = reset[0, 5] = reset[0, 6] = reset[0, 64] = reset[0, 127] = reset[0, 332] = True
    reset[1, 100:140] = True
    want = reference(v, 0.2, reset)
    got = device(v, 0.2, reset)
    compare(got, want, dtype, wide=size > 64)
    assert bool((got["d_log_decay"].cpu()[reset] == 0).all())


def test_every_step_a_reset():
    v = make(1, 70, 2, 2, 16, 16, torch.float32)
    reset = torch.ones(1, 70, dtype=torch.bool)
    compare(device(v, 0.2, reset), {k: w for k, w in reference(v, 0.2, reset).items() if k not in ("d_log_decay", "d_state")}, torch.float32)
    got = device(v, 0.2, reset)
    assert float(got["d_state"].abs().max()) == 0 and float(got["d_log_decay"].abs().max()) == 0


@pytest.mark.parametrize("with_state, grads", [(False, ("grad", "grad_last")), (True, ("grad",)), (True, ("grad_last",)), (False, ("grad",))])
@pytest.mark.parametrize("steps", [40, 500])
def test_parts_left_out(steps, with_state, grads):
    v = make(2, steps, 2, 1, 24, 40, torch.float32)
    want = reference(v, 0.2, with_state=with_state, grads=grads)
    got = device(v, 0.2, with_state=with_state, grads=grads)
    for name in list(want):
        if want[name] is None:   # (nothing of it reaches the gradient)
            assert float(got[name].abs().max()) == 0
            del want[name]
    compare(got, want, torch.float32)


@pytest.mark.parametrize("decay", [0.0, -1e-6, -3.0, -50.0, -1e4, -float("inf"), 0.05])
def test_decays_of_all_sizes(decay):
    v = make(1, 150, 1, 1, 16, 16, torch.float32)
    v["log_decay"][:, 20:60] = decay
    v["log_decay"][:, 100] = decay
    want = reference(v, 0.2)
    if decay == -float("inf"):
        # (the definition's derivative is exp(-inf) times something: zero)
        want["d_log_decay"] = torch.nan_to_num(want["d_log_decay"])
    # exp(0.05 x 40): sums that grow carry the same relative error
    compare(device(v, 0.2), want, torch.float32)


def test_small_gradients_of_strong_decays():
    """The gradient of a decay of e^-15 is e^-15 of the others' size and keeps its own bits."""
    v = make(1, 128, 1, 1, 16, 16, torch.float32)
    v["log_decay"].fill_(-15.0)
    want, got = reference(v, 0.2)["d_log_decay"], device(v, 0.2)["d_log_decay"].double().cpu()
    assert float(((got - want).abs() / want.abs().max()).max()) < 1e-5


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides(dtype):
    v = make(2, 150, 4, 4, 20, 20, dtype)
    want = reference(v, 0.2)
    # one projection's parts, heads in front of steps, sequences that share their decays and queries' rows
    fused = torch.cat([v[k] for k in ("q", "k", "v")], -1).cuda()
    q, k, x = (t.detach().requires_grad_() for t in fused.split(20, -1))
    ld = v["log_decay"].cuda().transpose(1, 2).contiguous().transpose(1, 2).requires_grad_()
    grad = v["grad"].cuda().permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    state = v["state"].cuda().transpose(2, 3).contiguous().transpose(2, 3).requires_grad_()
    o, last = tb.linear_attention(q, k, x, ld, state, scale=0.2)
    d = torch.autograd.grad([o, last], [q, k, x, ld, state], [grad, v["grad_last"].cuda()])
    got = dict(zip(("o", "last", "d_q", "d_k", "d_v", "d_log_decay", "d_state"), (o, last, *d)))
    compare(got, want, dtype)
    # rows of odd addresses; expanded inputs
    buffer = torch.zeros(2 * 150 * 4 * 20 + 1, dtype=dtype, device="cuda")
    buffer[1:] = v["k"].cuda().flatten()
    o2, _ = tb.linear_attention(q.detach(), buffer[1:].view(2, 150, 4, 20), x.detach(), ld.detach(), state.detach(), scale=0.2)
    assert torch.equal(o2, o.detach())
    per_head = torch.tensor([-0.1, -0.2, -0.3, 0.0], device="cuda", requires_grad=True)
    one = v["q"].cuda()[:1, :, :1].expand(2, 150, 4, 20)
    o3, _ = tb.linear_attention(one, k.detach(), x.detach(), per_head.expand(2, 150, 4), scale=0.2)
    w = {**v, "q": one.cpu(), "log_decay": per_head.detach().cpu().expand(2, 150, 4).contiguous(), "state": torch.zeros_like(v["state"])}
    ref = reference(w, 0.2, grads=("grad",))
    assert float((o3.double().cpu() - ref["o"]).abs().max() / ref["o"].abs().max()) <= tolerance("o", dtype, False)
    d_decay, = torch.autograd.grad(o3, per_head, grad)
    want_decay = ref["d_log_decay"].sum((0, 1))
    # (300 terms of either sign, each to the tolerance of the largest)
    assert float((d_decay.double().cpu() - want_decay).abs().max() / ref["d_log_decay"].abs().max()) <= 300 * tolerance("d_log_decay", dtype, False)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("where", ["q", "k", "v", "grad", "state", "log_decay"])
def test_what_is_not_finite_stays_where_it_is(where, dtype):
    """One bad step in the middle of a chunk: steps in front of it and other documents do not see it."""
    v = make(1, 190, 2, 2, 20, 24, dtype)
    reset = torch.zeros(1, 190, dtype=torch.bool)
    reset[0, 80] = reset[0, 100] = True
    clean = device(v, 0.2, reset)
    for bad in (float("nan"), float("inf")):
        w = {k: t.clone() for k, t in v.items()}
        if where == "state":
            w["state"][0, 0] = bad
        else:
            w[where][0, 90, 0] = bad
        got = device(w, 0.2, reset)
        # forward: from the bad step to its document's end; a bad state up to the first reset
        seen = torch.zeros(190, dtype=torch.bool)
        if where == "state":
            seen[:80] = True
        elif where == "q":
            seen[90] = True
        elif where != "grad":
            seen[90:100] = True
        o = got["o"][0].cpu()
        assert torch.equal(o[~seen], clean["o"][0].cpu()[~seen]) or float((o[~seen].double() - clean["o"][0].cpu()[~seen].double()).abs().max()) <= \
            2 * tolerance("o", dtype, False) * float(clean["o"].abs().max())
        assert not bool(torch.isfinite(o[seen][:, 0].float()).all()) or not bool(seen.any())
        assert torch.isfinite(o[:, 1].float()).all()     # (the other head)
        assert torch.isfinite(got["last"]).all()
        # backward: other documents are as they were
        other = torch.ones(190, dtype=torch.bool)
        other[80:100] = False
        if where == "state":
            other[:80] = False
        for name in ("d_q", "d_k", "d_v", "d_log_decay"):
            a, b = got[name][0].cpu()[other].double(), clean[name][0].cpu()[other].double()
            assert torch.isfinite(a).all(), (where, name)
            assert float((a - b).abs().max()) <= 2 * tolerance(name, dtype, False) * float(clean[name].abs().max()), (where, name)
        if where in ("q", "k", "v", "grad"):
            assert torch.isfinite(got["d_state"]).all()
            # rows of the document that the bad one does not meet: q and grad reach back, k and v forward
            early, late = slice(80, 90), slice(91, 100)
            names = {"q": (("d_q", early), ("d_q", late), ("d_k", late), ("d_v", late)), "grad": (("d_q", early), ("d_q", late), ("d_k", late), ("d_v", late)),
                     "k": (("d_q", early), ("d_k", early), ("d_v", early), ("d_v", late)), "v": (("d_q", early), ("d_k", early), ("d_k", late), ("d_v", early))}
            for name, part in names[where]:
                a, b = got[name][0].cpu()[part].double(), clean[name][0].cpu()[part].double()
                assert float((a - b).abs().max()) <= 2 * tolerance(name, dtype, False) * float(clean[name].abs().max()), (where, name, part)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1), (3, 4, 2, 64, 64), (2, 6, 6, 100, 100), (5, 3, 1, 128, 77), (1, 2, 2, 5, 128), (64, 16, 16, 64, 64)])
def test_steps(shape, dtype):
    batch, heads, groups, features, values = shape
    v = make(batch, 4, heads, groups, features, values, dtype)
    want, last = [], None
    whole, last = tb.linear_attention(*(v[k].double() if k != "log_decay" else v[k].double() for k in NAMES))
    state = v["state"].cuda()
    address = state.data_ptr()
    for t in range(4):
        o = tb.linear_attention_step(*(v[k][:, t].cuda() for k in NAMES[:4]), state)
        # a sum of products of `features` numbers in 24 bits, rounded once
        tol = 1e-5 if dtype == torch.float32 else HALF
        assert o.dtype == dtype and float((o.cpu().double() - whole[:, t]).abs().max() / whole.abs().max()) <= tol
    assert state.data_ptr() == address
    assert float((state.cpu().double() - last).abs().max() / last.abs().max()) <= 1e-5


def test_steps_go_on_from_a_prompt():
    v = make(2, 100, 4, 2, 32, 48, torch.float32)
    c = {k: t.cuda() for k, t in v.items()}
    whole, last = tb.linear_attention(*(c[k] for k in NAMES))
    _, state = tb.linear_attention(*(c[k][:, :90] for k in NAMES[:4]), c["state"])
    for t in range(90, 100):
        o = tb.linear_attention_step(*(c[k][:, t] for k in NAMES[:4]), state)
        assert float((o - whole[:, t]).abs().max()) <= 1e-5 * float(whole.abs().max())
    assert float((state - last).abs().max()) <= 1e-5 * float(last.abs().max())


def test_nothing_to_do():
    for batch, steps, heads, groups in ((0, 5, 2, 2), (2, 0, 2, 1), (2, 5, 0, 0)):
        v = {k: t.cuda() for k, t in make(batch, steps, max(heads, 1), max(groups, 1), 8, 8, torch.float32).items()}
        if heads == 0:
            v = {k: t[:, :, :0] if t.dim() == 4 and k not in ("state", "grad_last") or k == "log_decay" else t[:, :0] for k, t in v.items()}
        leaves = [v[k].requires_grad_() for k in NAMES]
        o, last = tb.linear_attention(*leaves)
        assert o.shape == v["v"].shape and torch.equal(last, v["state"])
        d = torch.autograd.grad([o, last], leaves, [v["grad"], v["grad_last"]])
        assert all(g.shape == t.shape for g, t in zip(d, leaves)) and torch.equal(d[4], v["grad_last"])


def test_same_bits_at_every_call_and_on_other_streams():
    v = make(2, 600, 3, 1, 40, 64, torch.bfloat16)
    want = device(v, 0.2)
    stream = torch.cuda.Stream()
    for s in (torch.cuda.current_stream(), stream, stream):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got = device(v, 0.2)
        torch.cuda.synchronize()
        for k in want:
            assert torch.equal(got[k], want[k]), k


@pytest.mark.parametrize("dtype, size", [(torch.float32, 64), (torch.bfloat16, 64), (torch.float32, 128), (torch.bfloat16, 100)])
def test_a_full_chip(dtype, size):
    """256 workgroups of some twenty chunks, wavefronts at their own pace: the same bits at every call, and some heads
    against the definition."""
    v = make(16, 700, 16, 16, size, size, dtype)
    c = {k: t.cuda() for k, t in v.items()}
    leaves = [c[k].requires_grad_() for k in NAMES]
    first = None
    for _ in range(4):
        o, last = tb.linear_attention(*leaves, scale=0.2)
        got = [o.detach(), last.detach(), *torch.autograd.grad([o, last], leaves, [c["grad"], c["grad_last"]])]
        if first is None:
            first = got
        for a, b in zip(got, first):
            assert torch.equal(a, b)
    for b, h in ((0, 0), (5, 7), (15, 15)):
        one = {k: (t[b:b + 1, h:h + 1] if k in ("state", "grad_last") else t[b:b + 1, :, h:h + 1]) for k, t in v.items()}
        part = dict(zip(("o", "last", "d_q", "d_k", "d_v", "d_log_decay", "d_state"), first))
        part = {k: (t[b:b + 1, h:h + 1] if k in ("last", "d_state") else t[b:b + 1, :, h:h + 1]) for k, t in part.items()}
        compare(part, reference(one, 0.2), dtype, wide=size > 64)


def test_captured_calls():
    v = {k: t.cuda() for k, t in make(2, 400, 3, 1, 40, 64, torch.float32).items()}
    leaves = [v[k].requires_grad_() for k in NAMES]

    def step():
        o, last = tb.linear_attention(*leaves, scale=0.2)
        return [o.detach(), last.detach(), *torch.autograd.grad([o, last], leaves, [v["grad"], v["grad_last"]])]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = step()
        graphs.append((graph, out))
    for n in range(3):
        with torch.no_grad():
            for t in leaves:
                t.mul_(0.9)
        want = step()
        for graph, out in graphs:
            for t in out:
                t.zero_()
            graph.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            for a, b in zip(out, want):
                assert torch.equal(a, b), n


def test_refusals():
    v = {k: t.cuda() for k, t in make(2, 5, 4, 2, 8, 8, torch.float32).items()}
    args = [v[k] for k in NAMES]

    def refused(text, *a, step=False, **kw):
        with pytest.raises(RuntimeError, match=text):
            (tb.linear_attention_step if step else tb.linear_attention)(*a, **kw)

    refused("must have the same dtype", args[0].bfloat16(), *args[1:])
    refused("float32 and bfloat16", *(t.double() for t in args[:3]), args[3])
    refused("q and k must have shape", args[0][:, :4], *args[1:])
    refused("multiple", args[0][:, :, :1].expand(2, 5, 3, 8), args[1][:, :, :1].expand(2, 5, 3, 8), *args[2:])
    refused("log_decay must have shape", *args[:3], args[3][:, :, :2])
    refused("log_decay must be float32", *args[:3], args[3].double())
    refused("state must have shape", *args[:4], args[4][:1])
    refused("state must be float32", *args[:4], args[4].bfloat16())
    refused("reset must be bool", *args, torch.zeros(2, 5, device="cuda"))
    refused("reset must have shape", *args, torch.zeros(2, 4, dtype=torch.bool, device="cuda"))
    refused("1 to 128", torch.zeros(1, 2, 1, 129, device="cuda"), torch.zeros(1, 2, 1, 129, device="cuda"), torch.zeros(1, 2, 1, 8, device="cuda"),
            torch.zeros(1, 2, 1, device="cuda"))
    refused("on the device", args[0].cpu(), *args[1:])
    one = [t[:, 0].contiguous() for t in args[:4]] + [args[4]]
    refused("contiguous", *one[:4], args[4].transpose(2, 3), step=True)
    refused("no gradient", one[0].requires_grad_(), *one[1:], step=True)
    o, _ = tb.linear_attention(args[0].requires_grad_(), *args[1:])
    g, = torch.autograd.grad(o.sum(), args[0], create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(g.sum(), args[0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("scale", [-0.4, 0.0])
def test_scales_of_any_sign(scale, dtype):
    v = make(2, 150, 2, 1, 40, 24, dtype)
    reset = torch.zeros(2, 150, dtype=torch.bool)
    reset[1, 70] = True
    compare(device(v, scale, reset), reference(v, scale, reset), dtype)


def test_states_at_any_address():
    """One step of a state that does not start at 16 bytes, and of one that does."""
    v = make(3, 1, 2, 2, 8, 12, torch.float32)
    args = [v[k].cuda()[:, 0] for k in NAMES[:4]]
    room = torch.empty(3 * 2 * 8 * 12 + 1, device="cuda")
    want = reference(v, 0.5)
    for start in (0, 1):
        state = room[start:start + 3 * 2 * 8 * 12].view(3, 2, 8, 12).copy_(v["state"])
        o = tb.linear_attention_step(*args, state, 0.5)
        assert (o.cpu() - want["o"][:, 0]).abs().max() <= 1e-5 * want["o"].abs().max()
        assert (state.cpu() - want["last"]).abs().max() <= 1e-5 * want["last"].abs().max()
