"""The group norm's PyTorch form where a group lies far from zero."""

import pytest
import torch

from rnn_with_grm_amd import cuda_ops


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16])
@pytest.mark.parametrize("W", [3, 7, 24, 40, 45, 128, 600, 4096])
def test_equal_values_leave_nothing(W, dtype):
    """What the first mean leaves of equal values is a few steps of them, the same of each, whose sum is exact: so is the second."""
    g = torch.Generator().manual_seed(W)
    values = torch.cat([torch.tensor([0.1, 777.7, -1e-3, 123456.7], dtype=torch.float64), 1000 * torch.rand(60, generator=g, dtype=torch.float64)])
    x = values.to(dtype)[:, None].expand(-1, 2 * W).contiguous()
    assert not cuda_ops.cuda_group_norm(x, 2).any()
