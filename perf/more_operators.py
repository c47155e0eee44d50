"""Operators of a sequence model with attention-like mixing and of its answers, as measurable cases.

A case is one pass through an operator: its forward call (serving, evaluation), or its forward call and the gradients of
every floating input (``train``).  Kinds:

* ``rotary``: features of queries and keys turned by angles that grow with the token's position, the first ``rotated`` of
  each head (or all), in pairs of neighbours (``interleaved``) or of the two halves; ``scale`` above one: frequencies for
  contexts so many times as long, slow ones divided by it, fast ones left, a ramp between;
* ``attention``: linear attention with a decay for each head, S_t = a_t S_{t-1} + k_t^T v_t and o_t = scale q_t S_t, over
  whole sequences; ``token``: its form for one new token per sequence, which updates the state in place.  ``groups`` of
  heads share queries and keys; ``reset``: packed documents, S_{t-1} counts as zero where one starts;
* ``sample``: a token for each row of logits from one given random number: temperature, the ``top_k`` largest, of those the
  most likely ones that make up ``top_p``, of those the ones at least ``min_p`` times as likely as the likeliest.

Where ``own`` is false a pass is computed in plain tensor operations, in 32 bits, rounded once (angles, sums of logarithms and
cumulated probabilities in 64).
"""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
BASE = 10000.0
CONTEXT = 2048                                  # tokens that unscaled frequencies were made for
CHUNK = 128                                     # of the plain form's attention
MAX_TURNED = 16 * 2048 * 16 * 64                # elements of the largest rotary call
MAX_ATTENTION = 16 * 2048 * 16 * 64 * 64        # tokens x heads x features x values of the largest attention with gradients
MAX_STATE = 64 * 16 * 64 * 64                   # elements of the largest state of the token form
MAX_LOGITS = 256 * 131072


def listed():
    return [
        # serving: queries and keys of one new token for each of 64 sequences
        _rotary("rotary_token", 64, 1, 32, 64, "f32", train=False),
        # a training batch's queries and keys
        _rotary("rotary_2048_step", 16, 2048, 16, 64, "bf16"),
        # one long row of packed documents, neighbours as pairs, half of an odd-sized head, a context of 32 times the length
        _rotary("rotary_long_forward", 1, 65537, 10, 100, "f32", rotated=50, interleaved=True, scale=32.0, train=False),
        # serving: one new token for each of 64 sequences
        _attention("attention_token", 64, 1, 16, 64, 64, "f32", token=True),
        # the same for a single sequence: pure latency
        _attention("attention_one_token", 1, 1, 16, 64, 64, "bf16", token=True),
        # a training batch, half-width storage
        _attention("attention_2048_step", 16, 2048, 16, 64, 64, "bf16"),
        # full-width storage, as the butterfly layers compute; a length that is a multiple of nothing useful
        _attention("attention_1001_step", 8, 1001, 16, 64, 64, "f32"),
        # one long row of packed documents, heads of an odd size
        _attention("attention_long_step", 1, 65537, 10, 100, 100, "bf16", reset=True),
        # prompts of wide heads that share queries and keys in pairs
        _attention("attention_128_forward", 4, 4096, 8, 128, 128, "bf16", groups=4, train=False),
        # serving: one sequence's answer, every filter on
        _sample("sample_one_row", 1, 32768, "f32", top_k=50, top_p=0.9, min_p=0.02),
        # a batch of sequences, nucleus only, a vocabulary that is a multiple of nothing
        _sample("sample_30001", 64, 30001, "f32", top_p=0.95),
        # a large batch over a large vocabulary, half-width storage
        _sample("sample_131072", 256, 131072, "bf16", top_p=0.9),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(("rotary", "attention", "attention", "attention", "sample"))
    dtype = rng.choice(("f32", "bf16"))
    if kind == "rotary":
        heads, features = spread(1, 64), 2 * spread(8, 64)
        rotated = features if rng.random() < 0.6 else 2 * rng.randint(1, features // 2)
        tokens = spread(1, max(1, min(65537, MAX_TURNED // (heads * features))))
        batch = rng.choice([b for b in (1, 2, 3, 5, 8, 16, 33, 64) if b <= tokens])
        case = _rotary(None, batch, tokens // batch, heads, features, dtype, rotated=rotated, interleaved=rng.random() < 0.4,
                       scale=rng.choice((1.0, 1.0, 4.0, 32.0)), train=rng.random() < 0.5)
    elif kind == "attention":
        features, values = spread(16, 128), spread(16, 128)
        groups, shared = spread(1, 16), rng.choice((1, 1, 1, 2, 3, 4))
        heads, token = groups * shared, rng.random() < 0.25
        if token:
            batch = spread(1, max(1, min(256, MAX_STATE // (heads * features * values))))
            case = _attention(None, batch, 1, heads, features, values, dtype, groups=groups, token=True)
        else:
            room = MAX_ATTENTION // (heads * max(features, 64) * max(values, 64))
            tokens = spread(1, max(1, min(65537, room)))
            batch = rng.choice([b for b in (1, 1, 2, 3, 5, 8, 16, 33) if b <= tokens])
            case = _attention(None, batch, tokens // batch, heads, features, values, dtype, groups=groups,
                              reset=rng.random() < 0.4, train=rng.random() < 0.7)
    else:
        vocab = spread(1000, 131072)
        rows = spread(1, max(1, min(1024, MAX_LOGITS // vocab)))
        case = _sample(None, rows, vocab, dtype, top_k=rng.choice((0, 0, 1, 20, 50, 400)), top_p=rng.choice((1.0, 0.95, 0.9, 0.5)),
                       min_p=rng.choice((0.0, 0.0, 0.02, 0.1)), greedy=rng.random() < 0.2)
    del case["name"]
    return case


def _rotary(name, batch, steps, heads, features, dtype, rotated=None, interleaved=False, scale=1.0, train=True):
    return dict(name=name, kind="rotary", batch=batch, steps=steps, heads=heads, features=features, rotated=rotated or features,
                dtype=dtype, interleaved=interleaved, scale=scale, train=train)


def _attention(name, batch, steps, heads, features, values, dtype, groups=None, token=False, reset=False, train=True):
    return dict(name=name, kind="attention", batch=batch, steps=steps, heads=heads, groups=groups or heads, features=features,
                values=values, dtype=dtype, token=token, reset=reset, train=train and not token)


def _sample(name, rows, vocab, dtype, top_k=0, top_p=1.0, min_p=0.0, greedy=False):
    return dict(name=name, kind="sample", rows=rows, vocab=vocab, dtype=dtype, top_k=top_k, top_p=top_p, min_p=min_p, greedy=greedy,
                train=False)


def _frequencies(case):
    """(rotated / 2) angles a position, float64, and the factor that goes with the scaling."""
    pairs, scale = case["rotated"] // 2, case["scale"]
    plain = BASE ** (-torch.arange(pairs, dtype=torch.float64) * 2 / case["rotated"])
    if scale == 1.0:
        return plain, 1.0
    # full turns within the original context: 32 and more stay, one and fewer are divided
    turns = plain * CONTEXT / (2 * math.pi)
    stay = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
    return plain * stay + plain / scale * (1.0 - stay), 0.1 * math.log(scale) + 1.0


def prepare(case, seed):
    """Activations, states, logits and random numbers as a training or serving program holds them on the GPU."""
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype, train = DTYPES[case["dtype"]], case["train"]

    def randn(*shape, scale=1.0, shift=0.0, dtype=dtype):
        return torch.randn(*shape, device=DEVICE, generator=gen, dtype=torch.float32).mul_(scale).add_(shift).to(dtype)

    def rand(*shape, dtype=torch.float32):
        return torch.rand(*shape, device=DEVICE, generator=gen, dtype=dtype)

    state, wanted = {"case": dict(case)}, {}
    if case["kind"] == "rotary":
        batch, steps = case["batch"], case["steps"]
        frequencies, state["magnitude"] = _frequencies(case)
        state["frequencies"] = frequencies.to(DEVICE)
        # each sequence from a position of its own, the last ones at the end of the (scaled) context
        first = torch.randint(0, max(1, int(CONTEXT * case["scale"]) - steps), (batch, 1), device=DEVICE, generator=gen)
        state["positions"] = first + torch.arange(steps, device=DEVICE)
        wanted["x"] = randn(batch, steps, case["heads"], case["features"])
        if train:
            state["grad"] = randn(batch, steps, case["heads"], case["features"])
    elif case["kind"] == "attention":
        batch, heads, features, values = case["batch"], case["heads"], case["features"], case["values"]
        lead = (batch,) if case["token"] else (batch, case["steps"])
        wanted["q"], wanted["k"] = randn(*lead, case["groups"], features), randn(*lead, case["groups"], features)
        wanted["v"] = randn(*lead, heads, values)
        # heads that remember from some ten tokens to some thousand, each token a little more or less
        reach = torch.logspace(1, 3, heads, device=DEVICE)
        wanted["log_decay"] = -torch.exp(randn(*lead, heads, scale=0.5, dtype=torch.float32)) / reach
        wanted["state"] = randn(batch, heads, features, values, dtype=torch.float32)
        state["scale"] = features ** -0.5
        if case["reset"]:
            # packed documents of some 1000 tokens
            state["reset"] = rand(*lead) < 1e-3
        if train:
            state["grad"] = randn(*lead, heads, values)
            state["grad_state"] = randn(batch, heads, features, values, dtype=torch.float32)
    else:
        rows, vocab = case["rows"], case["vocab"]
        logits = randn(rows, vocab, scale=2.5)
        # a tenth is ruled out by a grammar, another one in each row
        state["logits"] = logits.masked_fill_(rand(rows, vocab) < 0.1, -math.inf)
        # every request has settings of its own around the case's
        temperature = 0.6 + 0.8 * rand(rows)
        if case["greedy"]:
            temperature = temperature.masked_fill(rand(rows) < 0.5, 0.0)
        state["temperature"] = temperature
        state["uniform"] = rand(rows)
        if case["top_k"]:
            state["top_k"] = torch.randint(1, 2 * case["top_k"] + 1, (rows,), device=DEVICE, generator=gen)
        if case["top_p"] < 1.0:
            state["top_p"] = case["top_p"] + (1.0 - case["top_p"]) * 0.5 * rand(rows)
        if case["min_p"] > 0.0:
            state["min_p"] = case["min_p"] * (0.5 + rand(rows))
    state["wanted"] = {k: v.requires_grad_(train) for k, v in wanted.items()}
    return state


def run(state):
    case = state["case"]
    if own:
        with torch.set_grad_enabled(case["train"]):
            return _run_own(state, case)
    with torch.no_grad():
        plain = {"rotary": _plain_rotary, "sample": _plain_sample,
                 "attention": _plain_token if case.get("token") else _plain_attention}[case["kind"]]
        return plain(state, case)


def _run_own(state, case):
    import butterfly_amd as tb
    w = state["wanted"]
    if case["kind"] == "sample":
        return tb.sample(state["logits"], state["uniform"], temperature=state["temperature"], top_k=state.get("top_k"),
                         top_p=state.get("top_p"), min_p=state.get("min_p"))
    if case["kind"] == "rotary":
        out = {"y": tb.rotary(w["x"], state["positions"], state["frequencies"], interleaved=case["interleaved"],
                              magnitude=state["magnitude"])}
        grads = {"y": "grad"}
    elif case["token"]:
        o = tb.linear_attention_step(w["q"], w["k"], w["v"], w["log_decay"], w["state"], scale=state["scale"])
        return {"o": o, "state": w["state"]}
    else:
        o, last = tb.linear_attention(w["q"], w["k"], w["v"], w["log_decay"], w["state"], state.get("reset"), scale=state["scale"])
        out, grads = {"o": o, "state": last}, {"o": "grad", "state": "grad_state"}
    if case["train"]:
        d = torch.autograd.grad([out[k] for k in grads], list(w.values()), [state[g] for g in grads.values()])
        out = {k: v.detach() for k, v in out.items()}
        out.update(("d_" + k, g) for k, g in zip(w, d))
    return out


# ---- the plain forms -------------------------------------------------------------------------------------

def _turn(x, cos, sin, rotated, interleaved):
    y = x.clone()
    part = x[..., :rotated]
    if interleaved:
        a, b = part[..., 0::2], part[..., 1::2]
        y[..., 0:rotated:2], y[..., 1:rotated:2] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = part[..., :rotated // 2], part[..., rotated // 2:]
        y[..., :rotated // 2], y[..., rotated // 2:rotated] = a * cos - b * sin, a * sin + b * cos
    return y


def _plain_rotary(state, case):
    dtype = DTYPES[case["dtype"]]
    angles = state["positions"].double().unsqueeze(-1) * state["frequencies"]
    cos = (torch.cos(angles) * state["magnitude"]).float().unsqueeze(-2)
    sin = (torch.sin(angles) * state["magnitude"]).float().unsqueeze(-2)
    out = {"y": _turn(state["wanted"]["x"].float(), cos, sin, case["rotated"], case["interleaved"]).to(dtype)}
    if case["train"]:
        out["d_x"] = _turn(state["grad"].float(), cos, -sin, case["rotated"], case["interleaved"]).to(dtype)
    return out


def _chunked(q, k, v, log_decay, first, reset):
    """(o, last) from (batch, steps, heads, ...) tensors in 32 bits: products of all pairs within chunks, a state from chunk to
    chunk."""
    batch, steps, heads, values = v.shape
    n = -(-steps // CHUNK)

    def cut(t):     # (batch, heads, chunks, CHUNK, ...), zeros behind the last step
        t = torch.cat((t, t.new_zeros(batch, n * CHUNK - steps, *t.shape[2:])), 1)
        return t.reshape(batch, n, CHUNK, *t.shape[2:]).movedim(3, 1).contiguous()

    q, k, v = cut(q), cut(k), cut(v)
    level = cut(log_decay).double().cumsum(3)
    if reset is None:
        part = torch.zeros_like(level, dtype=torch.int32)
    else:
        part = cut(reset.to(torch.int32).unsqueeze(-1).expand(batch, steps, heads)).cumsum(3)
    below = torch.ones(CHUNK, CHUNK, device=v.device).tril() > 0
    seen = below & (part.unsqueeze(-1) == part.unsqueeze(-2))
    decay = torch.exp((level.unsqueeze(-1) - level.unsqueeze(-2)).masked_fill(~seen, -math.inf).float())
    inside = torch.matmul(torch.matmul(q, k.transpose(-1, -2)) * decay, v)
    from_start = torch.exp(level.masked_fill(part != 0, -math.inf).float()).unsqueeze(-1)
    to_end = torch.exp((level[..., -1:] - level).masked_fill(part != part[..., -1:], -math.inf).float()).unsqueeze(-1)
    added = torch.matmul((k * to_end).transpose(-1, -2), v)
    s, starts = first, []
    for c in range(n):
        starts.append(s)
        s = s * from_start[:, :, c, -1:] + added[:, :, c]
    o = inside + torch.matmul(q * from_start, torch.stack(starts, 2))
    return o.movedim(1, 3).reshape(batch, n * CHUNK, heads, values)[:, :steps], s


def _plain_attention(state, case):
    w, dtype = state["wanted"], DTYPES[case["dtype"]]
    shared = case["heads"] // case["groups"]
    with torch.set_grad_enabled(case["train"]):
        leaves = [w[name].detach().float().requires_grad_(case["train"]) for name in ("q", "k", "v", "log_decay", "state")]
        q, k = (t.repeat_interleave(shared, 2) if shared > 1 else t for t in leaves[:2])
        o, last = _chunked(q * state["scale"], k, *leaves[2:], state.get("reset"))
        out = {"o": o.detach().to(dtype), "state": last.detach()}
        if case["train"]:
            d = torch.autograd.grad([o, last], leaves, [state["grad"].float(), state["grad_state"]])
            out.update(("d_" + name, g.to(w[name].dtype)) for name, g in zip(w, d))
    return out


def _plain_token(state, case):
    w, dtype = state["wanted"], DTYPES[case["dtype"]]
    shared = case["heads"] // case["groups"]
    q, k = (w[name].float().repeat_interleave(shared, 1) for name in "qk")
    s = w["state"]
    s.mul_(torch.exp(w["log_decay"])[..., None, None]).add_(k.unsqueeze(-1) * w["v"].float().unsqueeze(-2))
    o = (s * (q * state["scale"]).unsqueeze(-1)).sum(-2)
    return {"o": o.to(dtype), "state": s}


def _plain_sample(state, case):
    logits, rows, vocab = state["logits"], case["rows"], case["vocab"]
    temperature = state["temperature"].double().unsqueeze(1)
    order = torch.sort(logits, dim=1, descending=True, stable=True)[1]
    x = logits.double()
    top = x.amax(1, keepdim=True)
    w = torch.exp((x - top) / torch.where(temperature > 0, temperature, 1.0))
    # greedy: the first of the largest
    w = torch.where(temperature > 0, w, 0.0)
    greedy = order[:, 0]
    sorted_w = w.gather(1, order)
    keep = sorted_w > 0
    if "top_k" in state:
        keep = keep & (torch.arange(vocab, device=w.device) < state["top_k"].unsqueeze(1))
    if "top_p" in state:
        cumulated = torch.where(keep, sorted_w, 0.0).cumsum(1)
        before = torch.cat((torch.zeros_like(cumulated[:, :1]), cumulated[:, :-1]), 1)
        keep = keep & (before < state["top_p"].double().unsqueeze(1) * cumulated[:, -1:])
    if "min_p" in state:
        keep = keep & (sorted_w >= state["min_p"].double().unsqueeze(1))
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(keep, sorted_w, 0.0))
    cumulated = kept.cumsum(1)
    drawn = (cumulated <= state["uniform"].double().unsqueeze(1) * cumulated[:, -1:]).sum(1)
    return torch.where(temperature[:, 0] > 0, drawn, greedy)


# ---- what a pass cannot do without -------------------------------------------------------------------------

def work(case):
    """Bytes: each input once, each output once.  Flops: an addition, a multiplication, a comparison or a function
    value is one; attention is counted in its recurrent form."""
    size, train = {"f32": 4, "bf16": 2}[case["dtype"]], case["train"]
    if case["kind"] == "rotary":
        tokens, pairs = case["batch"] * case["steps"], case["rotated"] // 2
        n = tokens * case["heads"] * case["features"]
        passes = 2 if train else 1
        return {"bytes": passes * 2 * n * size + tokens * 8 + pairs * 8,
                "flops": passes * 6 * tokens * case["heads"] * pairs + 4 * tokens * pairs}
    if case["kind"] == "attention":
        tokens, heads = case["batch"] * case["steps"], case["heads"]
        square = case["features"] * case["values"]
        rows = tokens * (2 * case["groups"] * case["features"] + 2 * heads * case["values"]) * size + tokens * heads * 4
        states = 2 * case["batch"] * heads * square * 4
        more = tokens if case["reset"] else 0
        if train:
            # again with o's gradient in o's place, and the gradients
            return {"bytes": 3 * rows - tokens * heads * case["values"] * size + 2 * states + more,
                    "flops": 15 * tokens * heads * square}
        return {"bytes": rows + states + more, "flops": 5 * tokens * heads * square}
    n = case["rows"] * case["vocab"]
    return {"bytes": n * size + case["rows"] * (16 + 8 * (case["top_k"] > 0) + 4 * (case["top_p"] < 1) + 4 * (case["min_p"] > 0)),
            "flops": 5 * n}


# ---- the same in 64 bits, from the definitions ---------------------------------------------------------------

def exact(case, seed):
    with torch.no_grad():
        state = prepare(case, seed)
        if case["kind"] == "sample":
            return _exact_sample(case, state)
        wide = {k: v.detach().double() for k, v in state["wanted"].items()}
        for k in ("grad", "grad_state"):
            if k in state:
                wide[k] = state[k].double()
        return (_exact_rotary if case["kind"] == "rotary" else _exact_attention)(case, state, wide)


def _exact_rotary(case, state, v):
    rotated = case["rotated"]
    pairs = torch.arange(rotated // 2, device=DEVICE)
    one, two = (2 * pairs, 2 * pairs + 1) if case["interleaved"] else (pairs, pairs + rotated // 2)
    turn = torch.polar(torch.full((), state["magnitude"], dtype=torch.float64, device=DEVICE),
                       torch.einsum("bt,p->btp", state["positions"].double(), state["frequencies"]))[:, :, None]

    def turned(x, by):
        z = torch.complex(x[..., one], x[..., two]) * by
        y = x.clone()
        y[..., one], y[..., two] = z.real, z.imag
        return y

    out = {"y": turned(v["x"], turn)}
    if case["train"]:
        out["d_x"] = turned(v["grad"], turn.conj())
    return out


def _exact_attention(case, state, v):
    """Step by step; the gradients from a second walk back over the steps."""
    if case["token"]:
        v = {k: t if k == "state" else t.unsqueeze(1) for k, t in v.items()}
    batch, steps, heads = v["log_decay"].shape
    which = torch.arange(heads, device=DEVICE) // (heads // case["groups"])
    q, k = v["q"][:, :, which] * state["scale"], v["k"][:, :, which]
    a = torch.exp(v["log_decay"])
    if case["reset"]:
        a = a * (~state["reset"]).double().unsqueeze(-1)
    s, o, dq = v["state"].clone(), torch.empty_like(v["v"]), torch.empty_like(q)
    for t in range(steps):
        s *= a[:, t, :, None, None]
        s += k[:, t, :, :, None] * v["v"][:, t, :, None, :]
        o[:, t] = torch.matmul(q[:, t, :, None], s)[:, :, 0]
        if case["train"]:
            dq[:, t] = torch.matmul(s, v["grad"][:, t, :, :, None])[..., 0]
    if case["token"]:
        return {"o": o[:, 0], "state": s}
    out = {"o": o, "state": s}
    if not case["train"]:
        return out
    e, dk, dv = v["grad_state"].clone(), torch.empty_like(k), torch.empty_like(v["v"])
    for t in range(steps - 1, -1, -1):
        e += q[:, t, :, :, None] * v["grad"][:, t, :, None, :]
        dk[:, t] = torch.matmul(e, v["v"][:, t, :, :, None])[..., 0]
        dv[:, t] = torch.matmul(k[:, t, :, None], e)[:, :, 0]
        e *= a[:, t, :, None, None]
    # what a step's factor scales is what later steps read of it, less what they wrote themselves
    through = (o * v["grad"]).sum(-1) - (v["v"] * dv).sum(-1)
    behind = (s * v["grad_state"]).sum((-1, -2))
    d_log = through.flip(1).cumsum(1).flip(1) + behind.unsqueeze(1)
    if case["reset"]:
        # counted from each document's own end
        last = state["reset"].flip(1).to(torch.int64)
        later = (last.cumsum(1) - last).flip(1)
        total = torch.cat((d_log, torch.zeros_like(d_log[:, :1])), 1)
        start = torch.where(state["reset"], torch.arange(steps, device=DEVICE), steps)
        following = torch.cummin(start.flip(1), 1)[0].flip(1)
        following = torch.cat((following[:, 1:], torch.full_like(following[:, :1], steps)), 1)
        d_log = torch.where((later > 0).unsqueeze(-1), d_log - total.gather(1, following.unsqueeze(-1).expand_as(d_log)), d_log)
        d_log = torch.where(state["reset"].unsqueeze(-1), 0.0, d_log)

    def summed(t):
        return t.reshape(batch, steps, case["groups"], -1, case["features"]).sum(3)

    return out | {"d_q": summed(dq) * state["scale"], "d_k": summed(dk), "d_v": dv, "d_log_decay": d_log, "d_state": e}


def _exact_sample(case, state):
    """Row by row on the host."""
    logits, uniform = state["logits"].double().cpu().numpy(), state["uniform"].double().cpu().numpy()
    temperature = state["temperature"].double().cpu().numpy()
    settings = {name: state[name].cpu().numpy() for name in ("top_k", "top_p", "min_p") if name in state}
    tokens = np.empty(case["rows"], np.int64)
    for r, row in enumerate(logits):
        if temperature[r] == 0:
            tokens[r] = row.argmax()
            continue
        ranked = np.argsort(-row, kind="stable")
        if "top_k" in settings:
            ranked = ranked[:settings["top_k"][r]]
        p = np.exp((row[ranked] - row[ranked[0]]) / temperature[r])
        if "top_p" in settings:
            running = np.cumsum(p)
            number = 1 + np.searchsorted(running[:-1], float(settings["top_p"][r]) * running[-1], side="left")
            ranked, p = ranked[:number], p[:number]
        if "min_p" in settings:
            likely = p >= float(settings["min_p"][r])
            ranked, p = ranked[likely], p[likely]
        by_index = np.argsort(ranked)
        ranked, running = ranked[by_index], np.cumsum(p[by_index])
        tokens[r] = ranked[np.searchsorted(running, uniform[r] * running[-1], side="right")]
    return torch.from_numpy(tokens).to(DEVICE)
