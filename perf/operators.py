"""The operators that stand next to butterfly layers in a sequence model, as measurable cases.

A case is one pass through an operator: its forward call (inference, evaluation), or its forward call
and the gradients of every floating input (``train``).  Kinds:

* ``norm``: layer norm;
* ``dropout``: ``residual + dropout(x)`` with a counter-based generator, alone or with the layer norm
  that follows it (``norm``);
* ``recurrence``: the gated linear recurrence over sequences, h_t = a_t h_{t-1} + (1 - a_t) x_t with
  a = sigmoid(gate), or h_t = a_t h_{t-1} + x_t with a = gate (``linear``); ``token``: its form for one
  new token per sequence, which updates the state in place;
* ``loss``: softmax cross entropy of ``hidden @ weight.T`` against targets, over a large vocabulary; the
  mean with its gradients in training, every row's own in evaluation.

Where ``own`` is false a pass is computed in plain tensor operations, in 32 bits, rounded once.
"""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "c64": torch.complex64}
EPS = 1e-5
IGNORE = -100
MAX_ELEMENTS = 32768 * 4096          # rows x columns of the largest norm
MAX_SEQUENCE = 16 * 2048 * 1024      # batch x steps x channels of the largest recurrence
MAX_PRODUCT = 8192 * 1024 * 32768    # rows x features x vocabulary of the largest loss
MAX_LOGITS = 8192 * 32768            # and its rows x vocabulary


def listed():
    return [
        # one decoding step of a small batch: pure latency
        _norm("norm_512_few_rows", 16, 512, "f32", train=False),
        # ragged rows and columns (a multiple of nothing useful), half-width storage
        _norm("norm_1000_step", 3001, 1000, "bf16"),
        # the widest rows at the largest training batch of the benchmark
        _norm("norm_4096_step", 32768, 4096, "f32"),
        # flattened images, a small batch, no residual
        _dropout("dropout_784_step", 50, 784, "f32", 0.5, residual=False),
        # a block's residual branch at the benchmark's batch
        _dropout("dropout_1024_step", 16384, 1024, "bf16", 0.1),
        # the same with the next block's norm behind it
        _dropout("dropout_norm_2048_step", 8192, 2048, "f32", 0.1, norm=True),
        # serving: one new token for each of 64 sequences
        _recurrence("recurrence_token", 64, 1, 1024, "f32", token=True),
        # a training batch of sequences
        _recurrence("recurrence_1024_step", 16, 2048, 1024, "f32"),
        # one long row of packed documents: few channels, many steps, neither a power of two
        _recurrence("recurrence_long_step", 1, 65537, 1000, "bf16", reset=True),
        # a training batch against a large vocabulary, half-width storage: the largest product
        _loss("loss_32768_step", 8192, 1024, 32768, "bf16"),
        # full-width storage, as the butterfly layers compute; no size a power of two
        _loss("loss_30001_step", 2000, 1000, 30001, "f32"),
        # evaluation of a short text with wide features
        _loss("loss_65536_forward", 512, 4096, 65536, "bf16", train=False),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(("norm", "dropout", "recurrence", "recurrence", "loss"))
    dtype = rng.choice(("f32", "bf16"))
    if kind in ("norm", "dropout"):
        cols = spread(32, 8192)
        rows = spread(1, max(1, min(32768, MAX_ELEMENTS // cols // (4 if kind == "dropout" else 1))))
        if kind == "norm":
            case = _norm(None, rows, cols, dtype, train=rng.random() < 0.7)
        else:
            residual = rng.random() < 0.7
            case = _dropout(None, rows, cols, dtype, rng.choice((0.0625, 0.1, 0.2, 0.5)), residual=residual,
                            norm=residual and rng.random() < 0.5, train=rng.random() < 0.8)
    elif kind == "recurrence":
        batch, cols = spread(1, 64), spread(16, 4096)
        if rng.random() < 0.2:
            case = _recurrence(None, batch, 1, cols, dtype, token=True, linear=rng.random() < 0.4)
        else:
            dtype = rng.choice(("f32", "f32", "bf16", "bf16", "c64"))
            steps = spread(1, max(1, min(65537, MAX_SEQUENCE // (batch * cols * (4 if dtype == "c64" else 1)))))
            case = _recurrence(None, batch, steps, cols, dtype, linear=dtype == "c64" or rng.random() < 0.3,
                               reset=rng.random() < 0.4, train=rng.random() < 0.7)
    else:
        features, vocab = spread(64, 4096), spread(1000, 131072)
        rows = spread(1, max(1, min(16384, MAX_LOGITS // vocab, MAX_PRODUCT // (features * vocab))))
        case = _loss(None, rows, features, vocab, dtype, train=rng.random() < 0.7)
    del case["name"]
    return case


def _norm(name, rows, cols, dtype, train=True):
    return dict(name=name, kind="norm", rows=rows, cols=cols, dtype=dtype, train=train)


def _dropout(name, rows, cols, dtype, p, residual=True, norm=False, train=True):
    return dict(name=name, kind="dropout", rows=rows, cols=cols, dtype=dtype, p=p, residual=residual, norm=norm, train=train)


def _recurrence(name, batch, steps, cols, dtype, token=False, linear=False, reset=False, train=True):
    return dict(name=name, kind="recurrence", batch=batch, steps=steps, cols=cols, dtype=dtype, token=token,
                linear=linear, reset=reset, train=train and not token)


def _loss(name, rows, features, vocab, dtype, train=True):
    return dict(name=name, kind="loss", rows=rows, features=features, vocab=vocab, dtype=dtype, train=train)


def prepare(case, seed):
    """Activations, parameters and output gradients as a training or serving program holds them on the GPU."""
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype, train = DTYPES[case["dtype"]], case["train"]

    def randn(*shape, scale=1.0, shift=0.0, dtype=dtype):
        wide = torch.complex64 if dtype.is_complex else torch.float32
        return torch.randn(*shape, device=DEVICE, generator=gen, dtype=wide).mul_(scale).add_(shift).to(dtype)

    state = {"case": dict(case)}
    if case["kind"] in ("norm", "dropout"):
        rows, cols = case["rows"], case["cols"]
        wanted = {"x": randn(rows, cols)}
        if case["kind"] == "dropout":
            # seed and call number
            state["rng"] = torch.randint(0, 1 << 62, (2,), device=DEVICE, generator=gen)
            if case["residual"]:
                wanted["residual"] = randn(rows, cols, scale=2.0)
        if case["kind"] == "norm" or case["norm"]:
            wanted["weight"] = randn(cols, scale=0.2, shift=1.0)
            wanted["bias"] = randn(cols, scale=0.2)
        if train:
            state["grad"] = randn(rows, cols)
            if case["kind"] == "dropout" and case["norm"]:
                state["grad_sum"] = randn(rows, cols)
    elif case["kind"] == "recurrence":
        batch, steps, cols = case["batch"], case["steps"], case["cols"]
        if case["token"]:
            wanted = {"gate": randn(batch, cols, shift=2.0), "x": randn(batch, cols)}
        else:
            wanted = {"gate": randn(batch, steps, cols, shift=2.0), "x": randn(batch, steps, cols)}
        if case["linear"]:
            # decay factors below one; complex ones turn too
            turn = torch.exp(1j * torch.pi * (wanted["gate"].imag)) if dtype.is_complex else 1.0
            wanted["gate"] = (torch.sigmoid(wanted["gate"].real.float()) * turn).to(dtype)
        full = torch.float32 if dtype == torch.bfloat16 else dtype
        wanted["state"] = randn(batch, cols, dtype=full)
        if case["reset"]:
            # packed documents of some 1000 tokens
            state["reset"] = torch.rand(batch, steps, device=DEVICE, generator=gen) < 1e-3
        if train:
            state["grad"] = randn(batch, steps, cols)
            state["grad_state"] = randn(batch, cols, dtype=full)
    else:
        rows, features, vocab = case["rows"], case["features"], case["vocab"]
        wanted = {"hidden": randn(rows, features), "weight": randn(vocab, features, scale=2.0 / features ** 0.5)}
        target = torch.randint(0, vocab, (rows,), device=DEVICE, generator=gen)
        # a tenth of the rows is padding; never all of them
        padding = torch.rand(rows, device=DEVICE, generator=gen) < 0.1
        padding[0] = False
        state["target"] = target.masked_fill(padding, IGNORE)
        if train:
            state["grad"] = randn(1, scale=0.1, shift=1.0, dtype=torch.float32)[0]
    state["wanted"] = {k: v.requires_grad_(train) for k, v in wanted.items()}
    return state


def run(state):
    case = state["case"]
    if own:
        with torch.set_grad_enabled(case["train"]):
            return _run_own(state, case)
    with torch.no_grad():
        plain = {"norm": _plain_norm, "dropout": _plain_dropout, "loss": _plain_loss,
                 "recurrence": _plain_token if case.get("token") else _plain_recurrence}[case["kind"]]
        return plain(state, case)


def _run_own(state, case):
    import butterfly_amd as tb
    w = state["wanted"]
    if case["kind"] == "norm":
        out = {"y": tb.layer_norm(w["x"], w["weight"], w["bias"], EPS)}
        grads = {"y": "grad"}
    elif case["kind"] == "dropout" and case["norm"]:
        y, total = tb.dropout_add_layer_norm(w["x"], state["rng"], case["p"], w["residual"], w["weight"], w["bias"], EPS)
        out, grads = {"y": y, "sum": total}, {"y": "grad", "sum": "grad_sum"}
    elif case["kind"] == "dropout":
        out = {"y": tb.dropout_add(w["x"], state["rng"], case["p"], w.get("residual"))}
        grads = {"y": "grad"}
    elif case["kind"] == "recurrence" and case["token"]:
        return {"h": tb.gated_recurrence_step(w["gate"], w["x"], w["state"], sigmoid=not case["linear"]), "state": w["state"]}
    elif case["kind"] == "recurrence":
        h, last = tb.gated_recurrence(w["gate"], w["x"], w["state"], state.get("reset"), sigmoid=not case["linear"])
        out, grads = {"h": h, "state": last}, {"h": "grad", "state": "grad_state"}
    else:
        out = {"loss": tb.linear_cross_entropy(w["hidden"], w["weight"], state["target"], ignore_index=IGNORE,
                                               reduction="mean" if case["train"] else "none")}
        grads = {"loss": "grad"}
    if case["train"]:
        d = torch.autograd.grad([out[k] for k in grads], list(w.values()), [state[g] for g in grads.values()])
        out = {k: v.detach() for k, v in out.items()}
        out.update(("d_" + k, g) for k, g in zip(w, d))
    return out


# ---- the plain forms -------------------------------------------------------------------------------------

def _norm_forward(x, weight, bias):
    centred = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt((centred * centred).mean(-1, keepdim=True) + EPS)
    unit = centred * r
    return unit * weight + bias, unit, r


def _norm_backward(g, unit, r, weight):
    gw = g * weight
    dx = r * (gw - gw.mean(-1, keepdim=True) - unit * (gw * unit).mean(-1, keepdim=True))
    return dx, (g * unit).sum(0), g.sum(0)


def _plain_norm(state, case):
    w, dtype = state["wanted"], DTYPES[case["dtype"]]
    y, unit, r = _norm_forward(w["x"].float(), w["weight"].float(), w["bias"].float())
    out = {"y": y}
    if case["train"]:
        out["d_x"], out["d_weight"], out["d_bias"] = _norm_backward(state["grad"].float(), unit, r, w["weight"].float())
    return {k: v.to(dtype) for k, v in out.items()}


def _times(a, m):
    """High and low 32 bits of a * m, a in 32 bits (held in 64), m < 2^32: by halves, so that nothing overflows."""
    low = (a & 0xFFFF) * m
    mid = (a >> 16) * m + (low >> 16)
    return mid >> 16, ((mid & 0xFFFF) << 16) | (low & 0xFFFF)


def _kept(rng, rows, cols, p):
    """Which elements stay: Philox4x32-10 with key rng[0] and counter (column // 8, row, rng[1]); element c of a
    row takes 16 bits, the low or high half of word (c % 8) // 2, and stays where they are >= round(65536 p)."""
    groups = -(-cols // 8)
    c0 = torch.arange(groups, device=rng.device).expand(rows, groups)
    c1 = torch.arange(rows, device=rng.device).unsqueeze(1).expand(rows, groups)
    c2, c3 = rng[1] & 0xFFFFFFFF, (rng[1] >> 32) & 0xFFFFFFFF
    c2, c3 = c2.expand(rows, groups), c3.expand(rows, groups)
    k0, k1 = rng[0] & 0xFFFFFFFF, (rng[0] >> 32) & 0xFFFFFFFF
    for _ in range(10):
        (h0, l0), (h1, l1) = _times(c0, 0xD2511F53), _times(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    words = torch.stack((c0, c1, c2, c3), -1)
    bits = torch.stack((words & 0xFFFF, words >> 16), -1).reshape(rows, groups * 8)[:, :cols]
    return bits >= round(65536 * p)


def _plain_dropout(state, case):
    w, dtype = state["wanted"], DTYPES[case["dtype"]]
    keep = _kept(state["rng"], case["rows"], case["cols"], case["p"])
    threshold = round(65536 * case["p"])
    scale = 65536 / (65536 - threshold) if threshold < 65536 else 0.0
    total = torch.where(keep, w["x"].float() * scale, 0.0)
    if case["residual"]:
        total = total + w["residual"].float()
    if case["norm"]:
        y, unit, r = _norm_forward(total, w["weight"].float(), w["bias"].float())
        out = {"y": y, "sum": total}
    else:
        out = {"y": total}
    if case["train"]:
        g = state["grad"].float()
        if case["norm"]:
            g, out["d_weight"], out["d_bias"] = _norm_backward(g, unit, r, w["weight"].float())
            g = g + state["grad_sum"].float()
        out["d_x"] = torch.where(keep, g * scale, 0.0)
        if case["residual"]:
            out["d_residual"] = g
    return {k: v.to(dtype) for k, v in out.items()}


def _scan(a, b, first):
    """h_t = a_t h_{t-1} + b_t from h_{-1} = first, by doubling: after each round (a, b) of step t stand for
    twice as many steps."""
    b = b.clone()
    b[:, 0] += a[:, 0] * first
    steps, reach = a.shape[1], 1
    while reach < steps:
        b = torch.cat((b[:, :reach], a[:, reach:] * b[:, :-reach] + b[:, reach:]), 1)
        a = torch.cat((a[:, :reach], a[:, reach:] * a[:, :-reach]), 1)
        reach *= 2
    return b


def _plain_recurrence(state, case):
    w, dtype = state["wanted"], DTYPES[case["dtype"]]
    full = torch.float32 if dtype == torch.bfloat16 else dtype
    gate, x, first = w["gate"].to(full), w["x"].to(full), w["state"]
    decay = gate if case["linear"] else torch.sigmoid(gate)
    into = x if case["linear"] else torch.sigmoid(-gate) * x
    carry = torch.where(state["reset"].unsqueeze(-1), 0.0, decay) if case["reset"] else decay
    h = _scan(carry, into, first)
    out = {"h": h.to(dtype), "state": h[:, -1].clone()}
    if case["train"]:
        # the same recurrence from the last step back: e_t = g_t + conj(a_{t+1}) e_{t+1}
        g = state["grad"].to(full).clone()
        g[:, -1] += state["grad_state"]
        back = torch.cat((torch.zeros_like(carry[:, :1]), carry[:, 1:].conj().flip(1)), 1)
        e = _scan(back, g.flip(1), torch.zeros_like(first)).flip(1)
        before = torch.cat((first.unsqueeze(1), h[:, :-1]), 1)
        if case["reset"]:
            before = torch.where(state["reset"].unsqueeze(-1), 0.0, before)
        if case["linear"]:
            d_gate, d_x = e * before.conj(), e
        else:
            rest = torch.sigmoid(-gate)
            d_gate, d_x = e * (before - x) * decay * rest, e * rest
        out |= {"d_gate": d_gate.to(dtype), "d_x": d_x.to(dtype), "d_state": carry[:, 0].conj() * e[:, 0]}
    return out


def _plain_token(state, case):
    w, dtype = state["wanted"], DTYPES[case["dtype"]]
    gate, x = w["gate"].float(), w["x"].float()
    decay = gate if case["linear"] else torch.sigmoid(gate)
    w["state"].copy_(decay * w["state"] + (x if case["linear"] else torch.sigmoid(-gate) * x))
    return {"h": w["state"].to(dtype), "state": w["state"]}


def _plain_loss(state, case):
    w, dtype, target = state["wanted"], DTYPES[case["dtype"]], state["target"]
    hidden, weight = w["hidden"].float(), w["weight"].float()
    logits = hidden @ weight.t()
    top = logits.amax(-1, keepdim=True)
    p = torch.exp(logits - top)
    sums = p.sum(-1, keepdim=True)
    counts = target != IGNORE
    at = target.clamp(min=0).unsqueeze(1)
    each = torch.log(sums) + top - logits.gather(1, at)
    each = torch.where(counts, each[:, 0], 0.0)
    out = {"loss": each}
    if case["train"]:
        number = counts.sum()
        out["loss"] = each.sum() / number
        p /= sums
        p.scatter_add_(1, at, torch.full_like(sums, -1.0))
        p *= torch.where(counts, state["grad"] / number, 0.0).unsqueeze(1)
        out |= {"d_hidden": (p @ weight).to(dtype), "d_weight": (p.t() @ hidden).to(dtype)}
    return out


# ---- what a pass cannot do without -------------------------------------------------------------------------

def work(case):
    """Bytes: each input once, each output once.  Flops: an addition, a multiplication, a comparison or a function
    value is one; the generator's integer operations are not counted."""
    size, train = {"f32": 4, "bf16": 2, "c64": 8}[case["dtype"]], case["train"]
    if case["kind"] in ("norm", "dropout"):
        n, norm = case["rows"] * case["cols"], case["kind"] == "norm" or case["norm"]
        tensors, flops = 2, 8 if norm else 0                    # x, y
        if train:
            tensors, flops = tensors + 2, flops + (14 if norm else 0)     # the gradients of both
        if case["kind"] == "dropout":
            flops += 4 if train else 2
            # the residual; the sum in front of a norm and, with gradients, the sum's and the residual's
            tensors += case["residual"] + case["norm"] * (3 if train else 1) + (case["residual"] and train and not case["norm"])
        return {"bytes": (tensors * n + (4 if train else 2) * norm * case["cols"]) * size, "flops": flops * n}
    if case["kind"] == "recurrence":
        n, full = case["batch"] * case["steps"] * case["cols"], max(size, 4)
        tensors, states = (6, 4) if train else (3, 2)
        flops = (2 if case["linear"] else 8) + ((4 if case["linear"] else 10) if train else 0)
        return {"bytes": tensors * n * size + states * case["batch"] * case["cols"] * full + case["reset"] * case["batch"] * case["steps"],
                "flops": flops * n * (4 if size == 8 else 1)}
    rows, features, vocab = case["rows"], case["features"], case["vocab"]
    operands = (rows + vocab) * features * size * (2 if train else 1)
    return {"bytes": operands + rows * (8 if train else 12), "flops": (6 if train else 2) * rows * features * vocab}


# ---- the same in 64 bits, from the definitions ---------------------------------------------------------------

def exact(case, seed):
    with torch.no_grad():
        state = prepare(case, seed)
        wide = {k: v.detach().to(torch.complex128 if v.is_complex() else torch.float64) for k, v in state["wanted"].items()}
        for k in ("grad", "grad_sum", "grad_state"):
            if k in state:
                wide[k] = state[k].to(torch.complex128 if state[k].is_complex() else torch.float64)
        if case["kind"] == "recurrence":
            return _exact_recurrence(case, state, wide)
        return {"norm": _exact_rows, "dropout": _exact_rows, "loss": _exact_loss}[case["kind"]](case, state, wide)


def _philox_bits(rng, rows, cols):
    """The 16-bit numbers of the generator, (rows, cols), in unsigned 64-bit arithmetic on the host."""
    seed, call = (int(v) & ((1 << 64) - 1) for v in rng.tolist())
    groups, word = (cols + 7) // 8, np.uint64(0xFFFFFFFF)
    counter = [np.tile(np.arange(groups, dtype=np.uint64), rows), np.repeat(np.arange(rows, dtype=np.uint64), groups),
               np.full(rows * groups, call & 0xFFFFFFFF, np.uint64), np.full(rows * groups, call >> 32, np.uint64)]
    key = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        first, third = counter[0] * np.uint64(0xD2511F53), counter[2] * np.uint64(0xCD9E8D57)
        counter = [(third >> np.uint64(32)) ^ counter[1] ^ np.uint64(key[0]), third & word,
                   (first >> np.uint64(32)) ^ counter[3] ^ np.uint64(key[1]), first & word]
        key = [(key[0] + 0x9E3779B9) & 0xFFFFFFFF, (key[1] + 0xBB67AE85) & 0xFFFFFFFF]
    halves = np.stack(counter, 1).astype("<u4").view("<u2").reshape(rows, groups * 8)
    return halves[:, :cols].astype(np.int32)


def _exact_rows(case, state, v):
    total, out = v["x"], {}
    if case["kind"] == "dropout":
        limit = int(math.floor(65536 * case["p"] + 0.5))
        bits = torch.from_numpy(_philox_bits(state["rng"], case["rows"], case["cols"])).to(DEVICE)
        factor = (bits >= limit).double() * (65536.0 / max(1, 65536 - limit))
        total = total * factor + v.get("residual", 0.0)
    normed = case["kind"] == "norm" or case["norm"]
    if normed:
        n = case["cols"]
        mean = total.sum(1) / n
        centred = total - mean[:, None]
        deviation = (centred.square().sum(1) / n + EPS).sqrt()
        unit = centred / deviation[:, None]
        out["y"] = torch.addcmul(v["bias"], unit, v["weight"])
        if case["kind"] == "dropout":
            out["sum"] = total
    else:
        out["y"] = total
    if case["train"]:
        g = v["grad"]
        if normed:
            out["d_weight"], out["d_bias"] = torch.einsum("rc,rc->c", g, unit), g.sum(0)
            g = g * v["weight"]
            g = (g - g.sum(1, keepdim=True) / n - unit * ((g * unit).sum(1, keepdim=True) / n)) / deviation[:, None]
        if case["kind"] == "dropout":
            g = g + v.get("grad_sum", 0.0)
            if case["residual"]:
                out["d_residual"] = g
            g = g * factor
        out["d_x"] = g
    return out


def _exact_recurrence(case, state, v):
    if case["token"]:
        v = {k: t.unsqueeze(1) if k in ("gate", "x") else t for k, t in v.items()}
    if case["steps"] > 200000:
        return None
    a = v["gate"] if case["linear"] else 1 / (1 + torch.exp(-v["gate"]))
    into = v["x"] if case["linear"] else v["x"] - a * v["x"]
    reset = state["reset"].unsqueeze(-1) if case["reset"] else None
    held = a if reset is None else a.masked_fill(reset, 0)
    h, before, now = torch.empty_like(into), torch.empty_like(into), v["state"]
    for t in range(case["steps"]):
        before[:, t] = now
        now = torch.addcmul(into[:, t], held[:, t], now)
        h[:, t] = now
    if case["token"]:
        return {"h": h[:, 0], "state": now}
    out = {"h": h, "state": now}
    if case["train"]:
        e, later = torch.empty_like(h), v["grad_state"]
        for t in range(case["steps"] - 1, -1, -1):
            e[:, t] = v["grad"][:, t] + later
            later = held[:, t].conj() * e[:, t]
        if reset is not None:
            before.masked_fill_(reset, 0)
        if case["linear"]:
            out |= {"d_gate": e * before.conj(), "d_x": e}
        else:
            out |= {"d_gate": e * (before - v["x"]) * a / (1 + torch.exp(v["gate"])), "d_x": e / (1 + torch.exp(v["gate"]))}
        out["d_state"] = later
    return out


def _exact_loss(case, state, v):
    target = state["target"]
    logits = torch.mm(v["hidden"], v["weight"].t())
    lse = torch.logsumexp(logits, 1)
    rows = torch.nonzero(target != IGNORE)[:, 0]
    picked = logits[rows, target[rows]]
    out = {"loss": torch.zeros_like(lse).index_copy_(0, rows, lse[rows] - picked)}
    if case["train"]:
        out["loss"] = out["loss"].sum() / len(rows)
        share = torch.zeros(case["rows"], dtype=torch.float64, device=DEVICE)
        share[rows] = v["grad"] / len(rows)
        d = logits.sub_(lse[:, None]).exp_()
        d[rows, target[rows]] -= 1
        d *= share[:, None]
        out |= {"d_hidden": torch.mm(d, v["weight"]), "d_weight": torch.mm(d.t(), v["hidden"])}
    return out
