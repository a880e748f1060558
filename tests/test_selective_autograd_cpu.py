"""Which calls of the selective scan and the short convolution ask for a derivative."""

import pytest
import torch
from torch.autograd import forward_ad

from rnn_with_grm_amd import cuda_ops


def test_a_tangent_is_a_wish_for_a_derivative():
    t, seen = torch.ones(3), []
    assert not cuda_ops._wants_grad(t, None)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(t, t)
        assert cuda_ops._wants_grad(None, dual) and not cuda_ops._wants_grad(t)
        with torch.no_grad():
            assert cuda_ops._wants_grad(dual)
    torch.func.jvp(lambda v: (seen.append(cuda_ops._wants_grad(v)), v)[1], (t,), (t,))
    assert seen == [True] and not cuda_ops._wants_grad(t)


def test_a_state_out_that_wants_a_gradient_is_refused():
    """It would be written behind autograd's back."""
    r = torch.randn
    with pytest.raises(ValueError, match="gradients are wanted"):
        cuda_ops.cuda_short_conv_step(r(2, 8), r(2, 3, 8), r(8, 4), state_out=r(2, 3, 8).requires_grad_())
    args = r(2, 1, 4), r(2, 2, 3), r(2, 1, 4), r(2, 2), -torch.ones(2), r(2, 2, 3, 4)
    out = r(2, 2, 3, 4).requires_grad_()
    with pytest.raises(ValueError, match="gradients are wanted"):
        cuda_ops.cuda_selective_step(*args, memory_out=out)
    with torch.no_grad():
        assert cuda_ops.cuda_selective_step(*args, memory_out=out)[1] is out
