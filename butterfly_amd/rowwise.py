"""What stands between two layers of a block: dropout, residual addition and layer norm, each row read once.

``layer_norm``, ``dropout_add`` and ``dropout_add_layer_norm`` (one kernel each way) with their modules.
Dropout is counter-based: ``rng`` is a tensor of two int64, a seed and the number of the call, and the mask is a
function of those, the row and the column (see ``dropout_mask``), made again in the backward pass instead
of stored.  Rows are float32 or bfloat16, of any width and row stride; ``weight`` and ``bias`` float32 or the
rows' dtype; statistics are formed in float32.  Host tensors run as tensor operations.  On the device the norms have no
second derivative (following a gradient's history raises), ``dropout_add`` has all of them.

No counterpart in the reference, whose users take these from PyTorch."""
import collections
import weakref

import torch
from torch import distributed as dist, nn

ops = torch.ops.torch_butterfly


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension."""
    if x.is_cuda:
        return ops.layer_norm(x, weight, bias, eps)
    return _host_norm(x, weight, bias, eps)


def dropout_add(x, rng, p, residual=None):
    """``residual + dropout(x)``: elements dropped with probability ``p`` (in steps of 1/65536), the others scaled by
    the inverse of the probability to stay.  A dropped element contributes zero whatever it is."""
    if x.is_cuda:
        return ops.dropout_add(x, rng, p, residual)
    return _host_total(x, rng, p, residual).to(x.dtype)


def dropout_add_layer_norm(x, rng, p, residual=None, weight=None, bias=None, eps=1e-5):
    """``(y, sum)`` with ``sum = residual + dropout(x)`` and ``y = layer_norm(sum)``."""
    if x.is_cuda:
        return ops.dropout_add_layer_norm(x, rng, p, residual, weight, bias, eps)
    total = _host_total(x, rng, p, residual)
    return _host_norm(total, weight, bias, eps).to(x.dtype), total.to(x.dtype)


def rng_next(rng, replica=0):
    """A copy of ``rng``, whose call number then goes up by one (on the device, in stream order: recorded in a HIP
    graph, every replay takes the next number).  ``replica``: which of several copies of a model that hold the same
    ``rng`` draws; each has a seed of its own."""
    if rng.is_cuda:
        return ops.rng_next(rng, replica)
    taken = rng.clone()
    # (2^64 over the golden ratio, modulo 2^64, as a signed number)
    taken[0] += (replica * 0x9E3779B97F4A7C15 + (1 << 63)) % (1 << 64) - (1 << 63)
    rng[1] += 1
    return taken


def dropout_mask(rng, rows, cols, p):
    """The elements that ``dropout_add`` keeps of (rows, cols), as bool, in plain tensor operations: Philox4x32-10 with
    key ``rng[0]`` and counter (column // 8, row, low and high half of ``rng[1]``) gives four 32-bit words for
    eight columns; column c takes the low (c even) or high 16 bits of word (c % 8) // 2 and is kept where they are
    at least ``round(65536 p)``."""
    groups, low = -(-cols // 8), 0xFFFFFFFF
    device = rng.device
    shape = (rows, groups)
    c = [torch.arange(groups, device=device).expand(shape), torch.arange(rows, device=device).unsqueeze(1).expand(shape),
         (rng[1] & low).expand(shape), (rng[1] >> 32 & low).expand(shape)]
    k = [rng[0] & low, rng[0] >> 32 & low]

    def product(a, m):   # (high, low) words of a * m, through halves of a
        mid = (a >> 16) * m + ((a & 0xFFFF) * m >> 16)
        return mid >> 16, a * (m & 0xFFFF) + ((a * (m >> 16) & 0xFFFF) << 16) & low

    for _ in range(10):
        (high0, low0), (high2, low2) = product(c[0], 0xD2511F53), product(c[2], 0xCD9E8D57)
        c = [high2 ^ c[1] ^ k[0], low2, high0 ^ c[3] ^ k[1], low0]
        k = [k[0] + 0x9E3779B9 & low, k[1] + 0xBB67AE85 & low]
    words = torch.stack(c, -1)
    return torch.stack((words & 0xFFFF, words >> 16), -1).reshape(rows, groups * 8)[:, :cols] >= round(65536 * p)


def _wide(x):
    return x if x.dtype == torch.float64 else x.float()


def _host_total(x, rng, p, residual):
    """In float where the device's kernels are, to be rounded once."""
    if not 0 <= p <= 1:
        raise ValueError(f"p must be between 0 and 1, got {p}")
    if p > 0 and rng is None:
        raise RuntimeError("dropout: p > 0 needs rng")
    threshold = round(65536 * p)
    total = _wide(x)
    if threshold > 0:
        keep = dropout_mask(rng, x.numel() // max(1, x.shape[-1]), x.shape[-1], p).reshape(x.shape)
        scale = 65536 / (65536 - threshold) if threshold < 65536 else 0.0
        total = torch.where(keep, total * scale, torch.zeros((), dtype=total.dtype))
    return total if residual is None else _wide(residual) + total


def _host_norm(x, weight, bias, eps):
    wide = _wide(x)
    centred = wide - wide.mean(-1, keepdim=True)
    y = centred * torch.rsqrt(centred.square().mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight
    if bias is not None:
        y = y + bias
    return y.to(x.dtype)


class LayerNorm(nn.Module):
    """``layer_norm`` over ``size`` features, with ``weight`` and ``bias`` (``elementwise_affine``) as ``nn.LayerNorm``
    names them."""

    def __init__(self, size, eps=1e-5, elementwise_affine=True, bias=True):
        super().__init__()
        self.size, self.eps = size, eps
        self.weight = nn.Parameter(torch.ones(size)) if elementwise_affine else None
        self.bias = nn.Parameter(torch.zeros(size)) if elementwise_affine and bias else None

    def forward(self, x):
        return layer_norm(x, self.weight, self.bias, self.eps)


# What forward calls drew that a backward pass may run again (torch.utils.checkpoint), by module and by a number from PyTorch's
# generator: the recomputation restores that generator, not a module's own, and so finds the number again.
_drawn = weakref.WeakKeyDictionary()
_DRAWN_AT_MOST = 1024       # of a module


def _may_run_again():
    """Whether somebody keeps the present call's inputs instead of what it saves: no gradient in training, or hooks on what
    is saved."""
    return not torch.is_grad_enabled() or torch._C._autograd._top_saved_tensors_default_hooks(False) is not None


class _Dropping(nn.Module):
    """Holds ``p`` and the generator's (seed, call), part of the state dict: a resumed run goes on where it stopped.

    ``replica``: the number of the model's copy that this process trains.  Copies on several GPUs hold the same ``rng``
    (``DistributedDataParallel`` sees to it, and a state dict that all of them load) and drop elements of their own by
    this number: by default the process's rank in ``torch.distributed``, where that is initialised.  Processes
    that work on the same activations give the same one.  A deep copy within a process drops what its original drops,
    until one of them is given another seed (``reseed``)."""

    def __init__(self, p, replica=None):
        super().__init__()
        if not 0 <= p <= 1:
            raise ValueError(f"p must be between 0 and 1, got {p}")
        self.p, self.replica = p, replica
        self.register_buffer("rng", torch.stack((torch.randint(1 << 62, ()), torch.zeros((), dtype=torch.int64))))

    def reseed(self, seed=None):
        """Another seed (by default one from PyTorch's generator), calls counted from zero."""
        seed = torch.randint(1 << 62, ()) if seed is None else torch.tensor(seed)
        self.rng.copy_(torch.stack((seed, torch.zeros_like(seed))))

    def _draw(self):
        """(rng of this call, p): nothing is dropped outside of training; a call that is run again draws what it drew."""
        if not self.training or self.p == 0:
            return None, 0.0
        again = torch._C._current_graph_task_id() != -1     # (a forward call inside of a backward pass)
        if not again and not _may_run_again():
            return self._next(), self.p
        calls, number = _drawn.setdefault(self, collections.OrderedDict()), int(torch.empty((), dtype=torch.int64).random_())
        if not again:
            calls[number] = self._next()
            if len(calls) > _DRAWN_AT_MOST:
                calls.popitem(last=False)
        elif number not in calls:
            raise RuntimeError("dropout: this forward call runs again inside of a backward pass and cannot tell which call it was: "
                               f"checkpoint with preserve_rng_state=True, at most {_DRAWN_AT_MOST} calls of a module at a time")
        return calls[number], self.p

    def _next(self):
        replica = self.replica
        if replica is None:
            replica = dist.get_rank() if dist.is_available() and dist.is_initialized() else 0
        return rng_next(self.rng, replica)


class DropoutAdd(_Dropping):
    """``residual + dropout(x)``, another mask at every call."""

    def forward(self, x, residual=None):
        rng, p = self._draw()
        return x if p == 0 and residual is None else dropout_add(x, rng, p, residual)


class DropoutAddLayerNorm(_Dropping):
    """``(layer_norm(sum), sum)`` with ``sum = residual + dropout(x)``: the end of one block and the norm of the next."""

    def __init__(self, size, p=0.1, eps=1e-5, replica=None):
        super().__init__(p, replica)
        self.size, self.eps = size, eps
        self.weight = nn.Parameter(torch.ones(size))
        self.bias = nn.Parameter(torch.zeros(size))

    def forward(self, x, residual=None):
        rng, p = self._draw()
        return dropout_add_layer_norm(x, rng, p, residual, self.weight, self.bias, self.eps)
