"""How far the selective scan's results are from its float64 definition beyond the outputs' own rounding.

``mag`` is the definition on magnitudes.  bfloat16 inputs: what a query reads of the state and the weights between
tokens are held as two bfloat16 parts, the second the rounded rest of the first, so 2^-8 * 2^-8 of a term is lost; the
float32 sums add the steps of the forward's own bound (N + 128 + T / 8 + 32) 2^-24."""

import pytest
import torch

import selective_oracle as oracle
from rnn_with_grm_amd import cuda_ops
from test_gpu_selective_bwd import magnitudes
from test_gpu_selective_scan import DTYPES, NAMES, U, definition, half, inputs, near, run

pytestmark = pytest.mark.gpu
PARTS = 2.0 ** -16 * 1.01


@pytest.mark.parametrize("B,T,H,P,G,N,lengths", [(2, 200, 4, 64, 2, 128, None), (2, 130, 3, 80, 1, 64, (130, 71)),
                                                 (1, 70, 2, 5, 1, 7, None), (1, 1100, 1, 64, 1, 96, None)])
def test_forward(dev, B, T, H, P, G, N, lengths):
    x = inputs(dev, B, T, H, P, G, N, torch.bfloat16, seed=T)
    n = None if lengths is None else torch.tensor(lengths, device=dev)
    hidden, memory = run(x, n)
    xr = dict(zip(NAMES, oracle.to64(*(x[k] for k in NAMES))))
    ref, rmem = definition(xr, n, True)
    mag, mmag = definition(xr, n, True, absolute=True)
    steps = N + 128 + T / 8 + 32
    near(hidden, ref, mag, torch.bfloat16, PARTS, steps)
    near(memory, rmem, mmag, torch.float32, 0, steps)


@pytest.mark.parametrize("dtype", DTYPES)
def test_an_infinity_stays_one(dev, dtype):
    """With positive keys and queries an infinite value, or element of the first state, is a sum that is infinite, with
    its sign, for its row of the state from its token on."""
    x = inputs(dev, 1, 150, 2, 32, 1, 32, dtype, seed=21)
    x["keys"], x["queries"], x["values"] = x["keys"].abs() + 0.125, x["queries"].abs() + 0.125, x["values"].clone()
    x["rates"] = x["rates"].clamp(min=-0.05)  # far from a decay of zero in float32
    x["values"][0, 20, 1, 5] = float("inf")
    x["memory"][0, 0, 9, 3] = float("-inf")
    hidden, memory = run(x)
    ref, rmem = definition(dict(zip(NAMES, oracle.to64(*(x[k] for k in NAMES)))), None, True)
    assert int((~torch.isfinite(ref)).sum()) == 130 + 150 and int((~torch.isfinite(rmem)).sum()) == 33
    for kind in (torch.isposinf, torch.isneginf, torch.isnan):  # (a NaN where a negative skip meets the infinite value)
        assert torch.equal(kind(hidden).cpu(), kind(ref)) and torch.equal(kind(memory).cpu(), kind(rmem))


@pytest.mark.parametrize("B,T,H,P,G,N,lengths", [(2, 200, 4, 64, 2, 128, None), (2, 130, 3, 80, 1, 64, (130, 71)),
                                                 (1, 70, 2, 5, 1, 7, None), (1, 1100, 1, 64, 1, 96, None)])
def test_gradients(dev, B, T, H, P, G, N, lengths):
    """The weights between tokens and the adjoint are two bfloat16 parts where keys, values and queries get their
    gradients from them; all else, the states in the step sizes' gradients among it, is float32 to its last bits: the
    bounds of test_gpu_selective_bwd without a rounding to 16 bits inside."""
    x = inputs(dev, B, T, H, P, G, N, torch.bfloat16, seed=T + 1)
    n = None if lengths is None else torch.tensor(lengths, device=dev)
    leaves = {k: x[k].detach().requires_grad_() for k in NAMES}
    outs = run(leaves, n)
    g = torch.Generator().manual_seed(T)
    dy, dm = torch.randn(outs[0].shape, generator=g).to(torch.bfloat16), torch.randn(outs[1].shape, generator=g)
    got = torch.autograd.grad(outs, [leaves[k] for k in NAMES], [dy.to(dev), dm.to(dev)])
    x64 = dict(zip(NAMES, oracle.to64(*(x[k] for k in NAMES), grad=True)))
    ref = oracle.selective_scan(*(x64[k] for k in NAMES), n, True)
    want = torch.autograd.grad(ref, [x64[k] for k in NAMES], (dy.double(), dm.double()))
    mags = magnitudes(x64, n, True, dy.double(), dm.double())
    steps = N + P + 256 + T / 8 + 64
    for k, a, b in zip(NAMES, got, want):
        try:
            near(a, b, mags[k], a.dtype, PARTS if k in ("keys", "values", "queries") else 0, steps)
        except AssertionError as e:
            raise AssertionError(f"gradient of {k}: {e}") from None


@pytest.mark.parametrize("bias,rate", [(-6.5, -12.0), (-4.5, -2.5)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_step_gradients_lean_to_no_side(dev, dtype, bias, rate):
    """Errors of the log decays' gradients dl_t of slow heads, whose keys, queries and values are mostly positive as a
    convolution with silu hands them over.  The gradients for `rates` and `step_bias` sum tens of thousands of them, so an
    error that leans to one side is seen there long before it is in any token's.  Blocks of 128 tokens are far enough apart
    to be independent but for the states they share: the sum over all blocks stays within 4 of its standard deviations
    (6e-5 of all inputs would not, were each block's error random)."""
    B, T, H, P, N = 8, 2048, 8, 64, 128
    g = torch.Generator(device=dev).manual_seed(31)
    r = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    x = {k: torch.nn.functional.silu(r(B, T, *s)).to(dtype) for k, s in (("keys", (1, N)), ("values", (H, P)), ("queries", (1, N)))}
    x.update(steps=r(B, T, H) * 0.5, rates=torch.full((H,), rate, device=dev), memory=0.2 * r(B, H, P, N), skip=r(H),
             step_bias=torch.full((H,), bias, device=dev))
    dy, dm = r(B, T, H, P).to(dtype), 0.1 * r(B, H, P, N)
    leaf = x["steps"].requires_grad_()
    (got,) = torch.autograd.grad(run(x), leaf, (dy, dm))
    x64 = {k: v.detach().double() for k, v in x.items()}
    leaf = x64["steps"].requires_grad_()
    plain = cuda_ops.cuda_selective_scan(*(x64[k] for k in NAMES[:6]), skip=x64["skip"], step_bias=x64["step_bias"],
                                         softplus=True, enabled=False)
    (want,) = torch.autograd.grad(plain, leaf, (dy.double(), dm.double()))
    slope = torch.sigmoid(x64["steps"].detach() + x64["step_bias"]) * x64["rates"]
    blocks = ((got.double() - want) / slope).unflatten(1, (T // 128, 128)).sum(2)
    lean = (blocks.sum() / blocks.square().sum().sqrt()).item()
    assert abs(lean) <= 4, f"{lean:.1f} standard deviations"
