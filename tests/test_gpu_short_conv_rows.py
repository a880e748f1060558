"""The short convolution's rows behind lengths, at the ends of runs and with values that are no numbers, against the
PyTorch form in float64 (held to the token-by-token definition by the CPU tests).  Tolerances as in test_gpu_short_conv."""

import math

import pytest
import torch

from rnn_with_grm_amd import cuda_ops
from test_gpu_short_conv import U, half, inputs

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def grads(x, w, b, st, silu, n, dy, ds):
    leaves = [t.detach().requires_grad_() for t in (x, w, b, st)]
    out = cuda_ops.cuda_short_conv(*leaves, activation="silu" if silu else None, lengths=n)
    return [*(o.detach() for o in out), *torch.autograd.grad(out, leaves, (dy, ds))]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C", [8, 5])
@pytest.mark.parametrize("W", [2, 3, 4])
def test_an_infinity_in_the_weights_gradient(dev, dtype, C, W):
    """Linear: x_t meets dy_t, ..., dy_{t + W - 1} in the weights' gradient, of which those behind the sequence do not
    exist.  Infinities in the last row of a sequence, in the last before a length and next to the ends of runs (16 tokens)."""
    x, w, b, st = inputs(dev, 2, 40, C, W, dtype, 3)
    n = torch.tensor([40, 21], device=dev)
    x = x.clone()
    x[0, 39, 0] = x[1, 20, 1] = float("inf")
    x[0, 15, 2], x[0, 16, 3] = float("inf"), float("-inf")
    g = torch.Generator().manual_seed(4)
    dy, ds = torch.randn(2, 40, C, generator=g).to(dtype).abs() + 0.125, torch.randn(2, W - 1, C, generator=g).to(dtype)
    got = grads(x, w, b, st, False, n, dy.to(dev), ds.to(dev))
    want = grads(*(t.double().cpu() for t in (x, w, b, st)), False, n.cpu(), dy.double(), ds.double())
    odd = torch.zeros(C, W, dtype=torch.bool)
    odd[:2, W - 1] = odd[2:4] = True
    assert torch.equal(torch.isinf(got[3]).cpu(), odd) and not torch.isnan(got[3]).any()
    full = torch.cat([st, x.masked_fill((torch.arange(40, device=dev) >= n[:, None])[..., None], 0)], 1).double().cpu()
    for i in range(W):  # the definition, sums of products that exist
        dw = torch.stack([sum((dy[s, t].double() * full[s, t + i]) for t in range(int(n[s]))) for s in range(2)]).sum(0)
        assert torch.equal(torch.isinf(dw), odd[:, i]) and torch.equal(got[3][odd[:, i], i].sign().cpu().double(), dw[odd[:, i]].sign())
    for i in (2, 4, 5):  # the gradients of x, the bias and the first state are finite, and x does not reach them
        assert torch.isfinite(got[i]).all() and torch.isfinite(want[i]).all()
