"""Tokens drawn from logits with given random numbers.

No counterpart in the reference."""
import torch

ops = torch.ops.torch_butterfly


def sample(logits, uniform, temperature=None, top_k=None, top_p=None, min_p=None):
    """A token (*), int64, for each row of ``logits`` (*, entries), float32 or bfloat16, from one random number of ``uniform``
    (*), float32 in [0, 1).

    With ``w = exp((logits - max) / temperature)``: of the ``top_k`` largest logits (ties: the lowest indexes) the
    likeliest ones until their sum reaches ``top_p`` of it (at least one), of those the ones with ``w >= min_p`` (at most 1); the
    token is the first index whose cumulated ``w``, in the order of indexes, exceeds ``uniform * total``.  Settings are
    a number for all rows or a tensor (*) (float32, ``top_k`` int64); ``None``, ``top_k <= 0``, ``top_p >= 1`` and
    ``min_p <= 0`` leave a filter out.  ``temperature <= 0``: the first of the largest logits; others count as between 2^-100 and 2^100.
    A setting that is NaN is none (a temperature: 0).

    NaN counts as -inf, and -inf is never drawn; a row of nothing else gives -1 (no index of anything).  Where +inf is among the logits, only those
    are drawn.  On the device weights are whole multiples of 2^-44 (the same token at every call), and up to
    2^19 entries are supported.  There is no gradient."""
    settings = [(temperature, 1.0, float), (top_k, 0, int), (top_p, 1.0, float), (min_p, 0.0, float)]
    if logits.is_cuda:
        args = []
        for value, default, kind in settings:
            tensor = isinstance(value, torch.Tensor)
            args += [value if tensor else None, default if tensor or value is None else kind(value)]
        return ops.sample(logits, uniform, *args)
    return _host_sample(logits, uniform, [default if value is None else value for value, default, _ in settings])


@torch.no_grad()
def _host_sample(logits, uniform, settings):
    lead, entries = logits.shape[:-1], logits.shape[-1]
    x = logits.reshape(-1, entries).to(torch.float64)
    x = torch.where(torch.isnan(x), -torch.inf, x) + 0.0
    temperature, top_k, top_p, min_p = (
        (s.reshape(-1) if isinstance(s, torch.Tensor) else torch.full((x.shape[0],), s, dtype=kind)).to(kind).unsqueeze(1)
        for s, kind in zip(settings, (torch.float64, torch.int64, torch.float64, torch.float64)))
    ordered, order = torch.sort(x, dim=1, descending=True, stable=True)
    greedy = ~(temperature > 0)
    w = torch.exp((ordered - ordered[:, :1]) / torch.where(greedy, 1.0, temperature).clamp(2.0 ** -100, 2.0 ** 100))
    w = torch.where(ordered == ordered[:, :1], 1.0, torch.where(ordered == -torch.inf, 0.0, w))
    w = torch.where(ordered[:, :1] == -torch.inf, 0.0, w)
    keep = (torch.arange(entries) < torch.where(top_k > 0, top_k, entries)) & (w > 0)
    before = torch.where(keep, w, 0.0).cumsum(1).roll(1, 1)
    total = before[:, :1].clone()
    before[:, 0] = 0.0
    keep &= (before < top_p.clamp(min=0.0) * total) | ~(top_p < 1.0)
    keep[:, 0] |= w[:, 0] > 0
    keep &= ~(w < min_p.clamp(max=1.0))
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0.0))
    running = kept.cumsum(1)
    u = torch.nan_to_num(uniform.reshape(-1, 1).to(torch.float64)).clamp(0.0, 1.0)
    token = (running <= u * running[:, -1:]).sum(1)
    # (a number of 1 draws the last entry that can be drawn)
    last = entries - 1 - (kept.flip(1) > 0).to(torch.int8).argmax(1)
    token = torch.where(greedy[:, 0], order[:, 0], torch.minimum(token, last))
    return torch.where(ordered[:, 0] == -torch.inf, -1, token).reshape(lead)
