"""The group norm of groups that lie far from zero.

The mean of a group is one float32 number; a second one, of what the first leaves, takes out what the first was off by."""

import pytest
import torch

import delta_oracle as oracle
from rnn_with_grm_amd import cuda_ops

pytestmark = pytest.mark.gpu
WIDTHS = [3, 7, 24, 40, 45, 128, 600, 2048, 4096]


@pytest.mark.parametrize("W", WIDTHS)
def test_equal_values_leave_nothing(dev, W):
    """The first mean of equal values x is off by a few steps of x at most: a number k steps of x, with k W below 2^24, whose
    sums are exact, so the second mean is that number and nothing is left."""
    g = torch.Generator().manual_seed(W)
    values = torch.cat([torch.tensor([0.1, 777.7, -1e-3, 123456.7]), 1000 * torch.rand(60, generator=g)])
    x = values.to(dev)[:, None].expand(-1, 2 * W).contiguous()
    assert not cuda_ops.cuda_group_norm(x, 2).any()
    leaf = x.clone().requires_grad_()
    weight = torch.ones(2 * W, device=dev, requires_grad=True)
    grads = torch.autograd.grad(cuda_ops.cuda_group_norm(leaf, 2, weight), (leaf, weight), torch.ones_like(x))
    assert not grads[1].any()  # (the sum of the normalised values)


@pytest.mark.parametrize("W", WIDTHS)
@pytest.mark.parametrize("offset", [100.0, -3000.0])
def test_a_mean_far_larger_than_the_deviation(dev, W, offset):
    """Values v = offset + noise, taken as they are in float32.  v less the first mean is rounded to half a step of |v|, but the
    first mean is a float32 number within a few steps of v, so the difference is a multiple of v's step (or of the mean's
    finer one) and exact wherever it is below 2^24 of them.  The second mean is off by (log2(W) + 64) half steps of
    the differences, at most 8 in size, over a deviation near one; the rest is the variance's and the root's, a few more:
    (log2(W) + 64) 2^-24 8 of unit rows, and the same of n for the variance, for which another n is counted."""
    g = torch.Generator().manual_seed(W)
    x = (offset + torch.randn(50, 2 * W, generator=g)).to(dev)
    got = cuda_ops.cuda_group_norm(x, 2).double().cpu()
    want = oracle.group_norm(x.double().cpu(), 2, None, None, None, False, True)
    r = 1 / torch.sqrt(x.double().cpu().view(50, 2, W).var(-1, unbiased=False, keepdim=True) + 1e-5)
    bound = ((torch.tensor(W).log2() + 64) * 2.0 ** -24 * 8 * (r + want.view(50, 2, W).abs())).flatten(1)
    assert ((got - want).abs() <= bound).all()
