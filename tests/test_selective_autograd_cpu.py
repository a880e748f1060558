"""Which calls of the selective scan and the short convolution ask for a derivative."""

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
