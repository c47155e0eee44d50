"""A linear layer onto a large vocabulary and its softmax cross entropy in one operator, the logits never held.

No counterpart in the reference."""
import torch
from torch import nn
from torch.nn import functional as F

_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


def linear_cross_entropy(hidden, weight, target, ignore_index=-100, reduction="mean"):
    """Cross entropy of ``hidden @ weight.T`` against ``target``: ``hidden`` (*, features), ``weight`` (vocabulary,
    features), ``target`` (*) int64, both float32 or both bfloat16; the loss is float32, (*) for ``reduction="none"``.

    Rows whose target is ``ignore_index`` count for nothing (the mean is over the others, NaN if there are none); a target
    that is no entry of the vocabulary makes loss and gradients NaN."""
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be 'none', 'mean' or 'sum', got {reduction!r}")
    if hidden.is_cuda:
        return torch.ops.torch_butterfly.linear_cross_entropy(hidden, weight, target, ignore_index, _REDUCTIONS[reduction])
    logits = F.linear(hidden, weight)
    logits = logits if logits.dtype == torch.float64 else logits.float()
    return F.cross_entropy(logits.flatten(0, -2), target.flatten(), ignore_index=ignore_index,
                           reduction=reduction).reshape(target.shape if reduction == "none" else ())


class LinearCrossEntropy(nn.Module):
    """The output layer of a language model together with its loss: ``weight`` (vocabulary, features)."""

    def __init__(self, features, vocabulary, ignore_index=-100, reduction="mean"):
        super().__init__()
        if reduction not in _REDUCTIONS:
            raise ValueError(f"reduction must be 'none', 'mean' or 'sum', got {reduction!r}")
        self.ignore_index, self.reduction = ignore_index, reduction
        self.weight = nn.Parameter(torch.randn(vocabulary, features) * features ** -0.5)

    def forward(self, hidden, target):
        return linear_cross_entropy(hidden, self.weight, target, self.ignore_index, self.reduction)
