"""The gated linear recurrence over sequences, channel by channel, for training and for one token at a time.

No counterpart in the reference."""
import torch

ops = torch.ops.torch_butterfly


def gated_recurrence(gate, x, state=None, reset=None, sigmoid=True):
    """``(h, last)`` with ``h[:, t] = a[:, t] * h[:, t-1] + b[:, t]`` from ``h[:, -1] = state`` (zeros by default), and
    ``last`` the state behind the last step.

    ``sigmoid``: ``a = sigmoid(gate)``, ``b = (1 - a) * x``; otherwise ``a = gate``, ``b = x``.  ``gate`` and ``x`` are
    (batch, steps, channels), float32, bfloat16 or (not sigmoid) complex64; states (batch, channels), float32 (complex64
    for complex rows).  ``reset`` (batch, steps), bool: there ``h[:, t-1]`` counts as zero (a packed document
    starts).  On the device there is no second derivative: following a gradient's history raises."""
    if x.is_cuda:
        return ops.gated_recurrence(gate, x, state, reset, sigmoid)
    wide = x.dtype if x.dtype.is_complex or x.dtype == torch.float64 else torch.float32
    a, b = _gates(gate.to(wide), x.to(wide), sigmoid)
    h = torch.zeros(x.shape[0], x.shape[2], dtype=wide) if state is None else state
    steps = []
    for t in range(x.shape[1]):
        decayed = a[:, t] * h
        if reset is not None:
            decayed = torch.where(reset[:, t, None], torch.zeros((), dtype=wide), decayed)
        h = decayed + b[:, t]
        steps.append(h)
    out = torch.stack(steps, 1) if steps else torch.zeros(x.shape, dtype=wide)
    return out.to(x.dtype), h.clone()


def gated_recurrence_step(gate, x, state, sigmoid=True):
    """One more step: ``state`` (batch, channels) is updated in place, the new ``h`` is returned in the dtype of ``x``
    (batch, channels).  For serving: no gradient."""
    if x.is_cuda:
        return ops.gated_recurrence_step(gate, x, state, sigmoid)
    if torch.is_grad_enabled() and any(t.requires_grad for t in (gate, x, state)):
        raise RuntimeError("gated_recurrence_step: has no gradient (use gated_recurrence, or torch.no_grad)")
    a, b = _gates(gate.to(state.dtype), x.to(state.dtype), sigmoid)
    state.copy_(a * state + b)
    return state.to(x.dtype, copy=True)


def _gates(gate, x, sigmoid):
    return (torch.sigmoid(gate), torch.sigmoid(-gate) * x) if sigmoid else (gate, x)
