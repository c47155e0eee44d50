"""A small language model whose projections are butterflies: embedding, blocks of a mixer (a gated recurrence or linear
attention with rotary positions) and a feed-forward part, a loss over the vocabulary, and tokens drawn from it.  It runs the
operators of ``rowwise``, ``recurrence``, ``attention``, ``positions``, ``loss`` and ``sampling`` together as a training or
serving program does."""
import torch
from torch import nn
from torch.nn import functional as F

from .attention import linear_attention, linear_attention_step
from .butterfly import Butterfly
from .loss import linear_cross_entropy
from .positions import rotary, rotary_frequencies
from .recurrence import gated_recurrence, gated_recurrence_step
from .rowwise import DropoutAddLayerNorm, LayerNorm, layer_norm
from .sampling import sample


class RecurrentMixer(nn.Module):
    """Gates and values from one ``Butterfly``, the recurrence over the steps, one ``Butterfly`` behind it."""

    def __init__(self, features, nblocks=1):
        super().__init__()
        self.into = Butterfly(features, 2 * features, nblocks=nblocks)
        self.out = Butterfly(features, features, nblocks=nblocks)

    def forward(self, x, state=None, reset=None):
        """(batch, steps, features) -> the same, and the state (batch, features) behind the last step."""
        gate, value = self.into(x).chunk(2, -1)
        h, last = gated_recurrence(gate, value, state, reset)
        return self.out(h), last

    def step(self, x, state):
        """(batch, features) of one more token; ``state`` is updated in place."""
        gate, value = self.into(x).chunk(2, -1)
        return self.out(gated_recurrence_step(gate, value, state))

    def empty_state(self, batch, device):
        return torch.zeros(batch, self.out.in_size, device=device)


class AttentionMixer(nn.Module):
    """Queries, keys, values and a decay for each head from one ``Butterfly``, positions, linear attention over the steps, each
    head's result normalised, one ``Butterfly`` behind it.  A state is the attention's and the next position of every sequence."""

    def __init__(self, features, heads, nblocks=1):
        super().__init__()
        if features % (2 * heads):
            raise ValueError(f"features must be a multiple of twice the heads, got {features} and {heads}")
        self.heads = heads
        self.into = Butterfly(features, 3 * features + heads, nblocks=nblocks)
        self.out = Butterfly(features, features, nblocks=nblocks)
        # (at first, heads that remember from some ten steps to some thousand)
        self.decay = nn.Parameter(torch.log(torch.logspace(1, 3, heads) - 1))
        self.register_buffer("frequencies", rotary_frequencies(features // heads)[0], persistent=False)

    def _apply(self, fn, recurse=True):
        # (the parameters' type is not the angles': a frequency of fewer than 64 bits loses them at far positions)
        frequencies = self.frequencies
        super()._apply(fn, recurse)
        if frequencies.is_meta:
            frequencies = rotary_frequencies(self.out.in_size // self.heads)[0]
        self.frequencies = frequencies.to(self.frequencies.device)
        return self

    def _parts(self, x, positions):
        """Queries and keys (turned), values, decays of x (*, features) at positions (*)."""
        features = self.out.in_size
        parts, decay = self.into(x).split((3 * features, self.heads), -1)
        parts = parts.reshape(*x.shape[:-1], 3 * self.heads, features // self.heads)
        q, k = rotary(parts[..., :2 * self.heads, :], positions, self.frequencies).split(self.heads, -2)
        return q, k, parts[..., 2 * self.heads:, :], F.logsigmoid(decay + self.decay)

    def forward(self, x, state=None, reset=None):
        """(batch, steps, features) -> the same, and the state behind the last step."""
        batch, steps = x.shape[:2]
        positions = torch.arange(steps, device=x.device).expand(batch, steps)
        matrix, first = (None, torch.zeros(batch, dtype=torch.int64, device=x.device)) if state is None else state
        o, last = linear_attention(*self._parts(x, positions + first.unsqueeze(1)), matrix, reset)
        return self.out(layer_norm(o).flatten(-2)), (last, first + steps)

    def step(self, x, state):
        """(batch, features) of one more token; ``state`` is updated in place."""
        matrix, positions = state
        o = linear_attention_step(*self._parts(x, positions), matrix)
        positions += 1
        return self.out(layer_norm(o).flatten(-2))

    def empty_state(self, batch, device):
        size = self.out.in_size // self.heads
        return torch.zeros(batch, self.heads, size, size, device=device), torch.zeros(batch, dtype=torch.int64, device=device)


class ButterflyLM(nn.Module):
    """``loss(tokens, target)`` for training, ``step(tokens, states)`` for one more token of every sequence, ``generate`` for
    some.  ``heads``: mixers of linear attention with that many heads (None: the gated recurrence)."""

    def __init__(self, vocabulary, features, layers, dropout=0.1, nblocks=1, heads=None):
        super().__init__()
        self.features = features
        self.embedding = nn.Parameter(torch.randn(vocabulary, features) * features ** -0.5)
        self.first_norm = LayerNorm(features)
        self.mixers = nn.ModuleList(RecurrentMixer(features, nblocks) if heads is None else AttentionMixer(features, heads, nblocks)
                                    for _ in range(layers))
        self.wide = nn.ModuleList(Butterfly(features, 2 * features, nblocks=nblocks) for _ in range(layers))
        self.narrow = nn.ModuleList(Butterfly(2 * features, features, nblocks=nblocks) for _ in range(layers))
        self.mixed = nn.ModuleList(DropoutAddLayerNorm(features, dropout) for _ in range(layers))
        self.fed = nn.ModuleList(DropoutAddLayerNorm(features, dropout) for _ in range(layers))

    def _blocks(self, tokens, mix):
        total = F.embedding(tokens, self.embedding)
        y = self.first_norm(total)
        for i in range(len(self.mixers)):
            y, total = self.mixed[i](mix(i, y), total)
            y, total = self.fed[i](self.narrow[i](F.gelu(self.wide[i](y))), total)
        return y

    def hidden(self, tokens, states=None, reset=None):
        """(batch, steps) tokens -> (batch, steps, features), and every layer's last state."""
        last = []

        def mix(i, y):
            out, state = self.mixers[i](y, None if states is None else states[i], reset)
            last.append(state)
            return out

        return self._blocks(tokens, mix), last

    def loss(self, tokens, target, reset=None, reduction="mean"):
        hidden, _ = self.hidden(tokens, reset=reset)
        return linear_cross_entropy(hidden, self.embedding, target, reduction=reduction)

    @torch.no_grad()
    def step(self, tokens, states):
        """(batch,) tokens -> logits (batch, vocabulary); ``states`` (one a layer) are updated in place."""
        y = self._blocks(tokens, lambda i, y: self.mixers[i].step(y, states[i]))
        return F.linear(y, self.embedding)

    @torch.no_grad()
    def generate(self, prompt, uniform, temperature=None, top_k=None, top_p=None, min_p=None):
        """(batch, prompt) tokens -> the (batch, steps) tokens that follow, drawn (as ``sample`` does) with ``uniform`` (batch,
        steps), random numbers in [0, 1).  Settings are numbers or one of each sequence.  Where nothing can be drawn (logits that are
        NaN or -inf, all of them) the token and those behind it are -1.  (Call ``eval()`` first: dropout.)"""
        hidden, states = self.hidden(prompt)
        logits, tokens = F.linear(hidden[:, -1], self.embedding), []
        for t in range(uniform.shape[1]):
            if t > 0:
                # (-1 is no row of the embedding: any row in its place, what comes of it is not looked at)
                logits = self.step(tokens[-1].clamp(min=0), states)
            token = sample(logits, uniform[:, t], temperature, top_k, top_p, min_p)
            tokens.append(torch.where(tokens[-1] < 0, tokens[-1], token) if tokens else token)
        return torch.stack(tokens, 1) if tokens else prompt[:, :0]

    def empty_states(self, batch):
        return [mixer.empty_state(batch, self.embedding.device) for mixer in self.mixers]
