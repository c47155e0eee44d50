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
    that is no entry of the vocabulary makes loss and gradients NaN.

    On the device sums are float32.  float32 operands of up to 64 rows (no more than features) are multiplied with 24
    bits; with more rows with 22 bits, which numbers (the probabilities of the backward pass among them) from 2^-28 of
    the operand's largest finite one up keep, and from 2^-40 up eleven.  Gradients of bfloat16 operands go through the logits'
    gradient in bfloat16.  There is no second derivative: following a gradient's history raises."""
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction must be 'none', 'mean' or 'sum', got {reduction!r}")
    if hidden.is_cuda:
        return torch.ops.torch_butterfly.linear_cross_entropy(hidden, weight, target, ignore_index, _REDUCTIONS[reduction])
    return _host_loss(hidden, weight, target, ignore_index, reduction)


def _host_loss(hidden, weight, target, ignore_index, reduction):
    wide = torch.float64 if hidden.dtype == torch.float64 else torch.float32
    logits, labels = F.linear(hidden.to(wide), weight.to(wide)).reshape(-1, weight.shape[0]), target.reshape(-1)
    wrong = (labels != ignore_index) & ((labels < 0) | (labels >= weight.shape[0]))
    if not wrong.any():
        loss = F.cross_entropy(logits, labels, ignore_index=ignore_index, reduction=reduction)
    else:
        # (any entry that counts, times NaN)
        loss = F.cross_entropy(logits, labels.masked_fill(wrong, int(ignore_index == 0)), ignore_index=ignore_index, reduction=reduction)
        loss = loss * (torch.where(wrong, torch.nan, 1.0).to(wide) if reduction == "none" else torch.nan)
    return loss.reshape(target.shape if reduction == "none" else ())


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
