"""Gradients of the selective state scan on the GPU against autograd through its float64 definition.

Tolerances.  Every gradient is a sum of products; ``mag`` is that sum with every term's magnitude, from
the definition on absolute values.  keys, values, queries, memory: as the outputs of the forward
(float32 arithmetic: (N + P + 2 * 128 + T / 8 + 64) 2^-24 of mag; bfloat16 inputs: weights and the adjoint rounded
once to bfloat16, half a step of mag; then half a step of the value).  The step sizes' gradient comes from
dl_t, the gradient of the log decay, a difference of sums over its block of at most 128 tokens: with
a_s = |dy_s . (h_s - D v_s)| and b_s = d_s |du_s . v_s| its float32 error is that many 2^-24 of the sum of a and b within
128 tokens and of |dl_t| itself; for bfloat16 inputs the states enter it with 16 bits, 2^-17 = 128 x 2^-24 more."""

import pytest
import torch

import selective_oracle as oracle
from rnn_with_grm_amd import cuda_ops
from test_gpu_selective_scan import DTYPES, NAMES, U, half, inputs, near, run

pytestmark = pytest.mark.gpu


def window(x, n=128):
    """Sum of [B, T, H] over the tokens within n of each."""
    T = x.shape[1]
    t = torch.arange(T)
    return torch.einsum("st,bth->bsh", ((t[:, None] - t[None]).abs() <= n).double(), x)


def magnitudes(x64, lengths, softplus, dy, dm):
    """The sums of magnitudes of every gradient, by NAMES."""
    v = {k: None if t is None else t.detach().nan_to_num() for k, t in x64.items()}
    B, T, H, P = v["values"].shape
    if lengths is not None:
        live = torch.arange(T) < torch.tensor(oracle.lengths_of(lengths, B, T))[:, None]
    else:
        live = torch.ones(B, T, dtype=torch.bool)
    z = v["steps"] if v["step_bias"] is None else v["steps"] + v["step_bias"]
    d = (torch.logaddexp(z, torch.zeros_like(z)) if softplus else z) * live[..., None]
    slope = torch.sigmoid(z) if softplus else torch.ones_like(z)
    rates = v["rates"].expand(B, T, H).clone().requires_grad_()
    leaf = {k: v[k].abs().requires_grad_() for k in ("keys", "values", "queries")}
    mem = None if v["memory"] is None else v["memory"].abs().requires_grad_()
    dl_leaf = d.clone().requires_grad_()
    h, m = oracle.selective_scan(leaf["keys"], leaf["values"], leaf["queries"], dl_leaf, rates, mem, None, None, lengths,
                                 False)
    outs = [leaf["keys"], leaf["values"], leaf["queries"], dl_leaf, rates] + ([mem] if mem is not None else [])
    grads = torch.autograd.grad((h, m), outs, (dy.abs(), dm.abs()), allow_unused=True)
    grads = [torch.zeros_like(o) if g is None else g for o, g in zip(outs, grads)]
    gk, gv, gq, gd, gr = grads[:5]
    dl = torch.where(d > 0, gr / d.clamp(min=1e-300), 0.0)
    direct = (gd - v["rates"] * dl) * live[..., None]
    near_dl = window((dy.abs() * h.detach()).sum(-1) + d * direct) + dl
    steps = (v["rates"].abs() * near_dl + direct) * slope * live[..., None]
    skip = (dy.abs() * leaf["values"].detach()).sum((0, 1, 3))
    gv = gv + (0 if v["skip"] is None else v["skip"].abs()[:, None] * dy.abs() * live[..., None, None])
    return {"keys": gk, "values": gv, "queries": gq, "steps": steps, "rates": (d * near_dl).sum((0, 1)),
            "memory": grads[5] if mem is not None else None, "skip": skip, "step_bias": steps.sum((0, 1))}


def check(dev, x, lengths, softplus, dtype, seed=5, parts=(True, True)):
    names = [k for k in NAMES if x[k] is not None]
    leaves = {k: (x[k].detach().requires_grad_() if k in names else None) for k in NAMES}
    hidden, memory = run(leaves, lengths, softplus)
    g = torch.Generator().manual_seed(seed)
    dy, dm = torch.randn(hidden.shape, generator=g).to(dtype), torch.randn(memory.shape, generator=g)
    outs = [o for o, on in zip((hidden, memory), parts) if on]
    ups = [u.to(dev) for u, on in zip((dy, dm), parts) if on]
    got = torch.autograd.grad(outs, [leaves[k] for k in names], ups)
    dy, dm = (u.double() * on for u, on in zip((dy, dm), parts))
    x64 = dict(zip(NAMES, oracle.to64(*(x[k] for k in NAMES), grad=True)))
    ref, rmem = oracle.selective_scan(*(x64[k] for k in NAMES), lengths, softplus)
    want = torch.autograd.grad((ref, rmem), [x64[k] for k in names], (dy, dm), allow_unused=True)
    mags = magnitudes(x64, lengths, softplus, dy, dm)
    B, T, H, P = x["values"].shape
    c = x["keys"].size(-1) + P + 256 + T / 8 + 64
    for k, gk, wk in zip(names, got, want):
        wk = torch.zeros_like(x64[k]) if wk is None else wk.nan_to_num()
        assert gk.dtype == x[k].dtype
        lossy = dtype == torch.bfloat16
        rounded = half(dtype) * 1.01 if lossy and k in ("keys", "values", "queries") else 0
        try:
            near(gk, wk, mags[k], gk.dtype, rounded, c + (128 if lossy else 0))
        except AssertionError as e:
            raise AssertionError(f"gradient of {k}: {e}") from None
    return got


CASES = [
    # B, T, H, P, G, N, lengths
    (1, 1, 1, 64, 1, 64, None), (2, 3, 2, 16, 1, 16, None), (1, 64, 2, 64, 1, 128, None), (2, 129, 4, 64, 2, 32, None),
    (1, 200, 2, 80, 1, 96, None), (3, 140, 2, 24, 2, 40, (0, 140, 33)), (1, 70, 3, 5, 1, 7, None),
    (2, 260, 2, 128, 1, 64, (260, 128)), (1, 128, 6, 32, 3, 128, None), (2, 0, 2, 16, 1, 16, None),
    (2, 90, 2, 33, 1, 24, (-4, 1000)),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,H,P,G,N,lengths", CASES)
def test_gradients(dev, B, T, H, P, G, N, lengths, dtype):
    x = inputs(dev, B, T, H, P, G, N, dtype, seed=T + P)
    n = None if lengths is None else torch.tensor(lengths, device=dev)
    if n is not None:
        dead = torch.arange(T, device=dev) >= n.clamp(0, T)[:, None]
        for k in ("keys", "values", "queries"):
            x[k] = x[k].masked_fill(dead[..., None, None], float("nan"))
    got = check(dev, x, n, True, dtype)
    if n is not None:
        for gk in got[:3]:
            assert (gk[dead] == 0).all()
        assert (got[3][dead] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_long_walk_in_parts(dev, dtype):
    x = inputs(dev, 2, 1100, 1, 16, 1, 24, dtype, seed=3)
    x["rates"] = x["rates"] * 0.05
    check(dev, x, torch.tensor([1100, 470], device=dev), True, dtype)


def test_one_output_only(dev):
    x = inputs(dev, 2, 100, 2, 32, 1, 32, torch.float32, seed=2)
    check(dev, x, None, True, torch.float32, parts=(True, False))
    check(dev, x, None, True, torch.float32, parts=(False, True))


def test_without_the_optional_inputs(dev):
    x = inputs(dev, 2, 100, 2, 32, 1, 32, torch.bfloat16, seed=4, steps_dtype=torch.float32)
    x["step_bias"], x["steps"] = x["step_bias"].abs(), x["steps"].abs() * 0.1
    for gone in (("memory",), ("skip",), ("step_bias",), ("memory", "skip", "step_bias")):
        check(dev, dict(x, **{k: None for k in gone}), None, False, torch.bfloat16)


def test_the_same_bits_twice(dev):
    x = inputs(dev, 2, 300, 4, 64, 1, 64, torch.bfloat16, seed=6)
    a, b = (check(dev, x, None, True, torch.bfloat16) for _ in range(2))
    assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_shared_and_expanded_inputs(dev):
    """Keys of one group serve all heads; a leaf expanded over the batch gets the batch's sum."""
    x = inputs(dev, 1, 80, 4, 16, 1, 16, torch.float32, seed=7)
    y = {k: (v if k in ("rates", "skip", "step_bias") else v.detach().requires_grad_()) for k, v in x.items()}
    wide = {k: (v if k in ("rates", "skip", "step_bias") else v.expand(3, *v.shape[1:])) for k, v in y.items()}
    names = ("keys", "values", "queries", "steps", "memory")
    a = torch.autograd.grad(run(wide)[0].sum(), [y[k] for k in names])
    b = torch.autograd.grad(run(y)[0].sum() * 3, [y[k] for k in names])
    for u, v in zip(a, b):
        torch.testing.assert_close(u, v, rtol=1e-5, atol=1e-5)


def test_against_differences(dev):
    """One directional derivative of the definition, by differences, against the kernels' gradients."""
    x = inputs(dev, 1, 70, 2, 16, 1, 16, torch.float32, seed=11)
    base = dict(zip(NAMES, oracle.to64(*(x[k] for k in NAMES))))
    g = torch.Generator().manual_seed(1)
    dirs = {k: torch.randn(v.shape, generator=g, dtype=torch.float64) for k, v in base.items()}
    dy = torch.randn(1, 70, 2, 16, generator=g, dtype=torch.float64)
    f = lambda h: (oracle.selective_scan(*(base[k] + h * dirs[k] for k in NAMES), None, True)[0] * dy).sum()  # noqa: E731
    slope = (f(1e-5) - f(-1e-5)) / 2e-5
    leaves = {k: v.detach().requires_grad_() for k, v in x.items()}
    grads = torch.autograd.grad(run(leaves)[0], [leaves[k] for k in NAMES], dy.float().to(dev))
    terms = [(a.double().cpu() * dirs[k]) for a, k in zip(grads, NAMES)]
    # float32 gradients, 512 steps of 2^-24 of the terms' magnitudes, and the differences' own 1e-8 or so.
    size = sum(t.abs().sum() for t in terms)
    assert abs(sum(t.sum() for t in terms) - slope) <= 512 * U * size + 1e-6


def test_step_under_autograd(dev):
    x = inputs(dev, 2, 1, 2, 16, 1, 16, torch.float32, seed=12)
    leaves = {k: v.detach().requires_grad_() for k, v in x.items()}
    args = [leaves[k][:, 0] for k in ("keys", "values", "queries", "steps")] + [leaves["rates"], leaves["memory"]]
    a = cuda_ops.cuda_selective_step(*args, skip=leaves["skip"], step_bias=leaves["step_bias"], softplus=True)
    b = run(leaves)
    assert torch.equal(a[0], b[0][:, 0]) and torch.equal(a[1], b[1])
    ga = torch.autograd.grad(a[0].sum() + a[1].sum(), [leaves[k] for k in NAMES])
    gb = torch.autograd.grad(b[0].sum() + b[1].sum(), [leaves[k] for k in NAMES])
    assert all(torch.equal(u, v) for u, v in zip(ga, gb))
