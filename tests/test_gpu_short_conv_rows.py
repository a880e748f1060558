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


def close(got, ref, mag, dtype, steps, what):
    got = got.double().cpu()
    assert got.shape == ref.shape
    bound = half(dtype) * ref.abs() * 1.001 + steps * U * mag + torch.finfo(dtype).smallest_normal * half(dtype) * 2
    bad = ~((got - ref).abs() <= bound)  # NaN is bad
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {((got - ref).abs() / bound).nan_to_num(99).max():.2f} of the bound"


def check(dev, B, T, C, W, silu, lengths, dtype, seed):
    x, w, b, st = inputs(dev, B, T, C, W, dtype, seed)
    n = None if lengths is None else torch.tensor(lengths, device=dev)
    dead = torch.zeros(B, T, dtype=torch.bool, device=dev) if n is None else torch.arange(T, device=dev) >= n.clamp(0, T)[:, None]
    clean = x.masked_fill(dead[..., None], 0.0)
    x = x.masked_fill(dead[..., None], float("nan"))  # not read
    g = torch.Generator().manual_seed(seed)
    dy, ds = torch.randn(B, T, C, generator=g).to(dtype), torch.randn(B, W - 1, C, generator=g).to(dtype)
    # The gradient of a dead row is not read either.
    got = grads(x, w, b, st, silu, n, dy.to(dev).masked_fill(dead[..., None], float("nan")), ds.to(dev))
    c = [t.double().cpu() for t in (clean, w, b, st)]
    nc = None if n is None else n.cpu()
    want = grads(*c, silu, nc, dy.double(), ds.double())
    # Magnitudes: the linear form on magnitudes, with silu's slope (at most 1.1, its own error half that of its argument).
    a = [t.abs() for t in c]
    pre = grads(*a, False, nc, dy.double().abs(), ds.double().abs())[0]
    rel = (1.1 + 0.5 * pre) if silu else 1.0
    mags = grads(*a, False, nc, dy.double().abs() * rel, ds.double().abs())
    mags[0] = pre * (1.1 if silu else 1.0)
    root = 16 * math.sqrt(max(B * T, 1))
    names = ("out", "state_out", "grad_x", "grad_weight", "grad_bias", "grad_state")
    for name, u, v, m, steps in zip(names, got, want, mags, (W + 11, 0, W + 16, root, root, W + 16)):
        close(u, v, m, dtype, steps, name)
    assert torch.equal(got[1].double().cpu(), want[1])
    assert (got[0][dead] == 0).all() and (got[2][dead] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,C,W,silu,lengths", [
    (3, 67, 72, 4, True, (67, 0, 5)), (2, 130, 7, 4, True, (1, 130)), (2, 40, 264, 2, False, (16, 17)), (3, 33, 40, 3, True, (1, 2, 31)),
    (4, 31, 128, 4, False, (-3, 2, 99, 31)), (2, 64, 33, 3, False, (63, 32)),
])
def test_rows_behind_the_lengths(dev, B, T, C, W, silu, lengths, dtype):
    """Neither x nor the output's gradient is read there; out and x's gradient are zeros."""
    check(dev, B, T, C, W, silu, lengths, dtype, T + C)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,C,W,lengths", [
    (3, 20011, 8, 4, None),           # runs of 21 tokens, no multiple of the four taken at once
    (3, 22501, 8, 3, None),           # 23, none of three
    (2, 29000, 5, 4, (29000, 12345)), # 20, element by element
    (3, 17000, 8, 2, (1, 17000, 16999)),
    (2, 1500, 5000, 4, None),         # 20 column blocks
])
def test_gradients_of_long_runs(dev, B, T, C, W, lengths, dtype):
    """As many rows as make the backward's runs longer than 16 tokens."""
    assert -(-B * T * -(-C // 256) // 3000) > 16
    check(dev, B, T, C, W, True, lengths, dtype, W)
