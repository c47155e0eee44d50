"""A small language model whose projections are butterflies: embedding, blocks of a gated recurrence and a feed-forward
part, and a loss over the vocabulary.  It runs the operators of ``rowwise``, ``recurrence`` and ``loss`` together as a
training or serving program does."""
import torch
from torch import nn
from torch.nn import functional as F

from .butterfly import Butterfly
from .loss import linear_cross_entropy
from .recurrence import gated_recurrence, gated_recurrence_step
from .rowwise import DropoutAddLayerNorm, LayerNorm


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


class ButterflyLM(nn.Module):
    """``loss(tokens, target)`` for training, ``step(tokens, states)`` for one more token of every sequence."""

    def __init__(self, vocabulary, features, layers, dropout=0.1, nblocks=1):
        super().__init__()
        self.features = features
        self.embedding = nn.Parameter(torch.randn(vocabulary, features) * features ** -0.5)
        self.first_norm = LayerNorm(features)
        self.mixers = nn.ModuleList(RecurrentMixer(features, nblocks) for _ in range(layers))
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

    def empty_states(self, batch):
        like = self.embedding
        return [torch.zeros(batch, self.features, device=like.device) for _ in self.mixers]
