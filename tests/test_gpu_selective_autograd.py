"""What the selective scan and the short convolution tell autograd."""

import pytest
import torch

from rnn_with_grm_amd import cuda_ops
from test_gpu_selective_scan import NAMES, inputs, run

pytestmark = pytest.mark.gpu


def test_the_first_state_may_be_moved_before_the_backward(dev):
    """The scan's backward does not read the first state, so a caller that keeps one buffer may overwrite it."""
    x = inputs(dev, 2, 70, 2, 16, 1, 16, torch.float32, seed=2)
    leaves = {k: (x[k] if k == "memory" else x[k].detach().requires_grad_()) for k in NAMES}
    names = [k for k in NAMES if k != "memory"]
    want = torch.autograd.grad(run(leaves)[0].sum(), [leaves[k] for k in names])
    hidden, memory = run(leaves)
    leaves["memory"].copy_(memory.detach())
    got = torch.autograd.grad(hidden.sum(), [leaves[k] for k in names])
    assert all(torch.equal(a, b) for a, b in zip(got, want))
