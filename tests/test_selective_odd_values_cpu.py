"""Infinities and NaN in the PyTorch forms of the selective scan and the short convolution: what reaches what."""

import pytest
import torch

from rnn_with_grm_amd import cuda_ops

INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("W", [2, 3, 4])
def test_an_infinity_before_a_length_in_the_weights_gradient(W):
    g = torch.Generator().manual_seed(1)
    x, w, st = torch.randn(1, 9, 3, generator=g), torch.randn(3, W, generator=g).requires_grad_(), torch.randn(1, W - 1, 3, generator=g)
    x[0, 5, 1] = INF
    out, _ = cuda_ops.cuda_short_conv(x, w, None, st, lengths=torch.tensor([6]))
    (dw,) = torch.autograd.grad(out.sum(), w)
    odd = torch.zeros(3, W, dtype=torch.bool)
    odd[1, W - 1] = True  # only its own token's gradient meets it
    assert torch.equal(torch.isinf(dw), odd) and not torch.isnan(dw).any()
