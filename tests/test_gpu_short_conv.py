"""Short causal convolution on the GPU against its float64 definition.

Tolerances.  A result is rounded once to its type (half a step: eps / 2 of the value).  Before that it
is a float32 sum of at most W + 1 products, so it is off by at most (W + 3) 2^-24 of the sum of the
products' magnitudes; silu has a slope of at most 1.1 and its exponential and reciprocal add 8
steps of 2^-24 of the value.  The weights' gradient sums n = B T products: its float32 sum is off by at most
n 2^-24 of the sum of the magnitudes (in random walk far less; 16 sqrt(n) is allowed)."""

import math

import pytest
import torch

import selective_oracle as oracle
from rnn_with_grm_amd import cuda_ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def half(dtype):
    return torch.finfo(dtype).eps / 2


def inputs(dev, B, T, C, W, dtype, seed, wide=True, state=True, wdtype=None):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x = r(B, T, C + 24).to(dtype).to(dev)[..., 8:8 + C] if wide else r(B, T, C).to(dtype).to(dev)
    wdtype = wdtype or dtype
    return (x, r(C, W).to(wdtype).to(dev) / 2, r(C).to(wdtype).to(dev) / 2,
            r(B, W - 1, C).to(dtype).to(dev) if state else None)


def near(got, ref, mag, dtype, steps):
    got, ref, mag = got.double().cpu(), ref.detach(), mag.detach()
    assert got.shape == ref.shape
    bound = half(dtype) * ref.abs() * 1.001 + steps * U * mag + torch.finfo(dtype).smallest_normal * half(dtype) * 2
    bad = (got - ref).abs() > bound
    assert not bad.any(), f"{int(bad.sum())} values off, worst {((got - ref).abs() / bound).max():.2f} of the bound"


CASES = [
    # B, T, C, W, silu, lengths
    (2, 1, 64, 4, True, None), (1, 2, 8, 3, True, None), (2, 3, 40, 2, False, None), (3, 67, 72, 4, True, (67, 0, 5)),
    (2, 130, 7, 4, True, (1, 130)), (1, 500, 33, 3, False, (499,)), (2, 64, 2304, 4, True, None),
    (4, 31, 128, 4, True, (-3, 2, 99, 31)), (2, 0, 16, 4, True, None), (33, 9, 264, 3, True, None),
]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,T,C,W,silu,lengths", CASES)
def test_forward_and_gradients(dev, B, T, C, W, silu, lengths, dtype):
    x, w, b, st = inputs(dev, B, T, C, W, dtype, seed=B * T + C)
    n = None if lengths is None else torch.tensor(lengths, device=dev)
    if n is not None:  # rows behind a length are not read
        dead = torch.arange(T, device=dev) >= n.clamp(0, T)[:, None]
        x = x.masked_fill(dead[..., None], float("nan"))
    leaves = [t.detach().requires_grad_() for t in (x, w, b, st)]
    out, state = cuda_ops.cuda_short_conv(*leaves, activation="silu" if silu else None, lengths=n)
    ref_in = oracle.to64(x, w, b, st, grad=True)
    ref, ref_state = oracle.short_conv(*ref_in, n, silu)
    with torch.no_grad():
        mag, _ = oracle.short_conv(*(t.nan_to_num().abs() for t in ref_in), n, False)
    near(out, ref, mag * 1.1, dtype, W + 11)
    assert torch.equal(state.double().cpu(), ref_state.detach())
    g = torch.Generator().manual_seed(5)
    dy, ds = (torch.randn(t.shape, generator=g).to(dtype) for t in (out, state))
    got = torch.autograd.grad((out, state), leaves, (dy.to(dev), ds.to(dev)))
    want = torch.autograd.grad((ref, ref_state), ref_in, (dy.double(), ds.double()), allow_unused=True)
    want = [torch.zeros_like(t) if v is None else v.nan_to_num() for t, v in zip(ref_in, want)]
    # Magnitudes of the gradients' sums: |dy| silu' <= 1.1 |dy|, whose own error is the slope's
    # (at most 0.5) times the error of pre, and 12 steps.
    with torch.no_grad():
        xa, wa, ba, sa = (t.nan_to_num().abs() for t in ref_in)
        rel = 1.1 + 0.5 * mag
        gmag = dy.double().abs() * rel
    def sums(g_):
        full = torch.cat([sa, xa], 1)
        live = torch.arange(T) < torch.tensor(oracle.lengths_of(n, B, T))[:, None]
        g_ = g_ * live[..., None]
        dfull = torch.zeros_like(full)
        dw = torch.zeros_like(wa)
        for i in range(W):
            dfull[:, i:i + T] += g_ * wa[:, i]
            dw[:, i] = (g_ * full[:, i:i + T]).sum((0, 1))
        return dfull[:, W - 1:] + ds.double().abs().amax(), dw, g_.sum((0, 1)), dfull[:, :W - 1] + ds.double().abs().amax()
    mags = sums(gmag)
    root = 16 * math.sqrt(max(B * T, 1))
    for got_, want_, mag_, steps in zip(got, want, mags, (W + 16, root, root, W + 16)):
        near(got_, want_, mag_, dtype, steps)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_float32_weights_of_a_16_bit_model(dev, dtype):
    x, w, b, st = inputs(dev, 2, 50, 48, 4, dtype, 3, wdtype=torch.float32)
    w.requires_grad_(), b.requires_grad_()
    out, state = cuda_ops.cuda_short_conv(x, w, b, st, activation="silu")
    ref_in = oracle.to64(x, w, b, st, grad=True)
    ref, _ = oracle.short_conv(*ref_in, None, True)
    with torch.no_grad():
        mag, _ = oracle.short_conv(*(t.abs() for t in ref_in), None, False)
    near(out, ref, mag * 1.1, dtype, 15)
    dw, db = torch.autograd.grad(out.float().sum(), (w, b))
    rw, rb = torch.autograd.grad(ref.sum(), ref_in[1:3])
    assert dw.dtype == db.dtype == torch.float32
    torch.testing.assert_close(dw.cpu().double(), rw, rtol=2e-5, atol=1e-4)
    torch.testing.assert_close(db.cpu().double(), rb, rtol=2e-5, atol=1e-4)


@pytest.mark.parametrize("missing", ["bias", "state", "both"])
def test_without_bias_or_state(dev, missing):
    x, w, b, st = inputs(dev, 2, 21, 24, 4, torch.float32, 9)
    b = None if missing in ("bias", "both") else b
    st = None if missing in ("state", "both") else st
    x.requires_grad_(), w.requires_grad_()
    out, state = cuda_ops.cuda_short_conv(x, w, b, st)
    ref_in = oracle.to64(x, w, b, st, grad=True)
    ref, ref_state = oracle.short_conv(*ref_in, None, False)
    torch.testing.assert_close(out.cpu().double(), ref.detach(), rtol=1e-5, atol=1e-5)
    assert torch.equal(state.cpu().double(), ref_state.detach())
    dx, dw = torch.autograd.grad(out.square().sum(), (x, w))
    rx, rw = torch.autograd.grad(ref.square().sum(), ref_in[:2])
    torch.testing.assert_close(dx.cpu().double(), rx, rtol=1e-5, atol=1e-5)
    torch.testing.assert_close(dw.cpu().double(), rw, rtol=1e-5, atol=1e-4)


def test_gradient_of_the_state_alone(dev):
    """A loss on the state that a call leaves reaches the last rows of x and the first state."""
    x, w, b, st = inputs(dev, 2, 2, 16, 4, torch.float32, 4)
    x.requires_grad_(), st.requires_grad_()
    _, state = cuda_ops.cuda_short_conv(x, w, b, st, activation="silu")
    dx, ds = torch.autograd.grad(state.sum(), (x, st))
    assert torch.equal(dx, torch.ones_like(dx))
    assert torch.equal(ds.cpu(), torch.tensor([0.0, 0.0, 1.0])[None, :, None].expand(2, 3, 16))


def test_gradient_against_differences(dev):
    x, w, b, st = (t.double().cpu() for t in inputs(dev, 1, 12, 8, 3, torch.float32, 12))
    g = torch.Generator().manual_seed(1)
    dirs = [torch.randn(t.shape, generator=g, dtype=torch.float64) for t in (x, w, b, st)]
    dy = torch.randn(1, 12, 8, generator=g, dtype=torch.float64)
    f = lambda h: (oracle.short_conv(*(t + h * d for t, d in zip((x, w, b, st), dirs)), None, True)[0] * dy).sum()  # noqa: E731
    slope = (f(1e-5) - f(-1e-5)) / 2e-5  # off by h^2 / 6 of the third derivative and 1e-16 / h: about 1e-9
    leaves = [t.float().to(dev).requires_grad_() for t in (x, w, b, st)]
    out, _ = cuda_ops.cuda_short_conv(*leaves, activation="silu")
    grads = torch.autograd.grad(out, leaves, dy.float().to(dev))
    got = sum((a.double().cpu() * d).sum() for a, d in zip(grads, dirs))
    size = sum((a.double().cpu() * d).abs().sum() for a, d in zip(grads, dirs))
    assert abs(got - slope) <= 64 * U * size


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,C,W", [(1, 8, 4), (3, 1000, 4), (2, 37, 3), (256, 64, 2)])
def test_step_continues_a_prompt(dev, B, C, W, dtype):
    """Token by token, in place and into a new state, as one call over the tokens does."""
    x, w, b, st = inputs(dev, B, 6, C, W, dtype, 2)
    out, state = cuda_ops.cuda_short_conv(x, w, b, st, activation="silu")
    kept, fresh = st.clone(), st
    for t in range(6):
        a, same = cuda_ops.cuda_short_conv_step(x[:, t], kept, w, b, activation="silu", state_out=kept)
        c, fresh = cuda_ops.cuda_short_conv_step(x[:, t], fresh, w, b, activation="silu")
        assert same is kept and torch.equal(a, c) and torch.equal(a, out[:, t])
    assert torch.equal(kept, state) and torch.equal(fresh, state)


def test_step_under_autograd(dev):
    x, w, b, st = inputs(dev, 2, 1, 16, 4, torch.float32, 7)
    w.requires_grad_()
    out, moved = cuda_ops.cuda_short_conv_step(x[:, 0], st, w, b, activation="silu")
    full, _ = cuda_ops.cuda_short_conv(x, w, b, st, activation="silu")
    assert torch.equal(out, full[:, 0])
    a, = torch.autograd.grad(out.sum(), w)
    c, = torch.autograd.grad(full.sum(), w)
    assert torch.equal(a, c)


def test_infinities_and_nan_reach_only_their_outputs(dev):
    x, w, b, st = inputs(dev, 1, 40, 8, 4, torch.float32, 8)
    x = x.clone()
    base, _ = cuda_ops.cuda_short_conv(x, w, b, st)
    x[0, 20, 3] = float("nan")
    x[0, 30, 5] = float("inf")
    out, _ = cuda_ops.cuda_short_conv(x, w, b, st)
    hit = torch.zeros(40, 8, dtype=torch.bool, device=dev)
    hit[20:24, 3] = True
    hit[30:34, 5] = True
    assert torch.equal(out[0][~hit], base[0][~hit])
    assert not torch.isfinite(out[0][hit]).any()


def test_expanded_batch_and_unaligned_rows(dev):
    """Strides of zero, and rows that no 16-byte access fits."""
    g = torch.Generator().manual_seed(6)
    x = torch.randn(1, 30, 19, generator=g).to(dev)[..., 1:17].expand(3, 30, 16)
    w, b = torch.randn(16, 4, generator=g).to(dev), torch.randn(16, generator=g).to(dev)
    out, state = cuda_ops.cuda_short_conv(x, w, b)
    want, wstate = cuda_ops.cuda_short_conv(x.contiguous().clone(), w, b)
    assert torch.equal(out, want) and torch.equal(state, wstate)
    leaf = torch.randn(1, 30, 16, generator=g).to(dev).requires_grad_()
    d, = torch.autograd.grad(cuda_ops.cuda_short_conv(leaf.expand(3, 30, 16), w, b)[0].sum(), leaf)
    e, = torch.autograd.grad(cuda_ops.cuda_short_conv(leaf, w, b)[0].sum() * 3, leaf)
    torch.testing.assert_close(d, e, rtol=1e-6, atol=1e-6)


def test_refusals(dev):
    x, w, b, st = inputs(dev, 2, 5, 16, 4, torch.float32, 1)
    conv, step = cuda_ops.cuda_short_conv, cuda_ops.cuda_short_conv_step
    for call in (lambda: conv(x, w[:, :1]), lambda: conv(x, torch.cat([w, w], 1)), lambda: conv(x, w[:8]),
                 lambda: conv(x, w, b[:3]), lambda: conv(x, w, b, st[:, :2]), lambda: conv(x, w, b, st.double()),
                 lambda: conv(x.double(), w.double()), lambda: conv(x, w.half()), lambda: conv(x, w, b.half()),
                 lambda: conv(x, w, lengths=torch.zeros(3, dtype=torch.long, device=dev)),
                 lambda: conv(x, w, lengths=torch.zeros(2, device=dev)),
                 lambda: conv(x, w, lengths=torch.zeros(2, dtype=torch.long)), lambda: conv(x, w.cpu()),
                 lambda: conv(x, w, activation="relu"), lambda: step(x, st, w), lambda: step(x[:, 0], st[:1], w),
                 lambda: step(x[:, 0], st, w, state_out=st[:, :, ::2]),
                 lambda: step(x[:, 0], st, w, state_out=st.half()),
                 lambda: step(x[:, 0], st, w.clone().requires_grad_(), state_out=st)):
        with pytest.raises(ValueError):
            call()
    both = torch.zeros(3, 3, 16, device=dev)
    with pytest.raises(RuntimeError):  # the new state half over the old one
        step(x[:, 0], both[:2], w, state_out=both[1:])


def test_captured_steps_and_prompts(dev):
    """A serving loop's step in place, and a prompt, replayed with other work between the replays."""
    x, w, b, st = inputs(dev, 4, 10, 64, 4, torch.bfloat16, 13)
    xs, kept = x[:, 0].clone(), st.clone()
    xp = x.contiguous()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cuda_ops.cuda_short_conv_step(xs, kept, w, b, activation="silu", state_out=kept)
        cuda_ops.cuda_short_conv(xp, w, b, st, activation="silu")
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = cuda_ops.cuda_short_conv_step(xs, kept, w, b, activation="silu", state_out=kept)
        pout, pstate = cuda_ops.cuda_short_conv(xp, w, b, st, activation="silu")
    kept.copy_(st)
    want, wstate = cuda_ops.cuda_short_conv(x, w, b, st, activation="silu")
    for t in range(10):
        xs.copy_(x[:, t])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[:, t])
        assert torch.equal(pout, want) and torch.equal(pstate, wstate)
        torch.randn(1000, 1000, device=dev).sum().item()
    assert torch.equal(kept, wstate)


def test_on_another_stream(dev):
    x, w, b, st = inputs(dev, 2, 300, 256, 4, torch.bfloat16, 14)
    want = cuda_ops.cuda_short_conv(x, w, b, st, activation="silu")
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = cuda_ops.cuda_short_conv(x, w, b, st, activation="silu")
    s.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
