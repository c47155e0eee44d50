"""Linear attention over heads that are not there."""
import pytest
import torch

import butterfly_amd as tb

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("steps", [0, 3, 700])
def test_queries_of_no_heads(steps, dtype):
    """Queries and keys of groups that no head of values uses: gradients of zeros."""
    q, k = (torch.randn(2, steps, 3, 8, device="cuda").to(dtype).requires_grad_() for _ in range(2))
    v = torch.zeros(2, steps, 0, 16, device="cuda", dtype=dtype, requires_grad=True)
    state = torch.zeros(2, 0, 8, 16, device="cuda", requires_grad=True)
    log_decay = torch.zeros(2, steps, 0, device="cuda", requires_grad=True)
    # (memory that the allocator gives out again)
    torch.full((2, steps, 3, 8), 7.0, device="cuda", dtype=dtype)
    o, last = tb.linear_attention(q, k, v, log_decay, state)
    assert o.shape == (2, steps, 0, 16) and last.shape == (2, 0, 8, 16)
    for leaf, d in zip((q, k, v, log_decay, state), torch.autograd.grad([o, last], [q, k, v, log_decay, state], [torch.zeros_like(o), torch.zeros_like(last)])):
        assert d.shape == leaf.shape and d.dtype == leaf.dtype and not bool(d.any())
