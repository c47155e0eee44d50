"""Linear attention with a decay for each head, for training and prompts and for one token at a time: the matrix-valued
sibling of ``gated_recurrence``.

No counterpart in the reference."""
import torch

ops = torch.ops.torch_butterfly


def linear_attention(q, k, v, log_decay, state=None, reset=None, scale=None):
    """``(o, last)`` with ``S[t] = exp(log_decay[t]) * S[t-1] + outer(k[t], v[t])`` from ``S[-1] = state`` (zeros by default),
    ``o[t] = scale * q[t] @ S[t]``, and ``last`` the state behind the last step, for each sequence and head.

    ``q``, ``k`` (batch, steps, groups, features), ``v`` (batch, steps, heads, values), all float32 or all bfloat16, heads of
    1 to 128 features and values; ``heads`` is a multiple of ``groups``, and ``heads / groups`` neighbouring heads share
    queries and keys.  ``log_decay`` (batch, steps, heads) float32; one of each head is ``decays.expand(batch, steps,
    heads)``.  States (batch, heads, features, values), float32.  ``reset`` (batch, steps), bool: there ``S[t-1]`` counts as
    zero (a packed document starts).  ``scale``: ``features ** -0.5`` by default.

    On the device sums and states are float32 (bfloat16: inner products that are factors again are rounded to 16 bits,
    results once to 8).  Decays below 2^-160 count as that, of 2^128 and more as infinite.  What is not finite (a decay, too) stays
    in its own document, and does not reach outputs and gradients of steps that do not meet it, except that gradients of
    ``log_decay`` are not finite for its whole document in the chunk of 64 (32) steps that holds it.  Decays above one that
    multiply up to 2^128 within a chunk are infinite there, and what they meet is infinite or NaN, zeros as well.  Training keeps
    a state for every chunk.  There is no second derivative: following a gradient's history raises."""
    if scale is None:
        scale = q.shape[-1] ** -0.5
    if v.is_cuda:
        return ops.linear_attention(q, k, v, log_decay, state, reset, scale)
    wide = _wide(v)
    shared = v.shape[2] // max(1, q.shape[2])
    q, k, x = q.to(wide).repeat_interleave(shared, 2), k.to(wide).repeat_interleave(shared, 2), v.to(wide)
    decay = torch.exp(log_decay.to(wide))[..., None, None]
    s = torch.zeros(v.shape[0], v.shape[2], q.shape[3], v.shape[3], dtype=wide) if state is None else state.to(wide)
    zero, steps = torch.zeros((), dtype=wide), []
    for t in range(v.shape[1]):
        decayed = decay[:, t] * s
        if reset is not None:
            decayed = torch.where(reset[:, t, None, None, None], zero, decayed)
        s = decayed + k[:, t].unsqueeze(-1) * x[:, t].unsqueeze(-2)
        steps.append(scale * (q[:, t].unsqueeze(-1) * s).sum(-2))
    out = torch.stack(steps, 1) if steps else torch.zeros(v.shape, dtype=wide)
    return out.to(v.dtype), s.clone()


def linear_attention_step(q, k, v, log_decay, state, scale=None):
    """One more step: ``state`` (batch, heads, features, values) is updated in place, the new ``o`` (batch, heads, values) is
    returned; ``q``, ``k`` (batch, groups, features), ``v`` (batch, heads, values), ``log_decay`` (batch, heads).  For
    serving: no gradient."""
    if scale is None:
        scale = q.shape[-1] ** -0.5
    if v.is_cuda:
        return ops.linear_attention_step(q, k, v, log_decay, state, scale)
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, log_decay, state)):
        raise RuntimeError("linear_attention_step: has no gradient (use linear_attention, or torch.no_grad)")
    shared = v.shape[1] // max(1, q.shape[1])
    wide = state.dtype
    q, k = q.to(wide).repeat_interleave(shared, 1), k.to(wide).repeat_interleave(shared, 1)
    state.mul_(torch.exp(log_decay.to(wide))[..., None, None]).add_(k.unsqueeze(-1) * v.to(wide).unsqueeze(-2))
    return (scale * (q.unsqueeze(-1) * state).sum(-2)).to(v.dtype)


def _wide(x):
    return torch.float64 if x.dtype == torch.float64 else torch.float32
