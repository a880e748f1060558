"""The short convolution and the selective scan as a layer runs them: one wide projection, the convolution over
values, keys and queries together, their slices into the scan, the prompt's states into single tokens; captured,
on several streams, over rows past 2^31 elements."""

import pytest
import torch

import selective_oracle as oracle
from rnn_with_grm_amd import cuda_ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def half(dtype):
    return torch.finfo(dtype).eps / 2


class Layer:
    """H heads of P values, G groups of N keys; x [B, T, H * P + 2 * G * N] and steps [B, T, H]."""

    def __init__(self, dev, dtype, B, T, H=4, P=32, G=2, N=32, W=4, seed=0):
        g = torch.Generator().manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
        self.shape, self.C, self.dtype = (H, P, G, N), H * P + 2 * G * N, dtype
        rows = r(B, T, self.C + H).to(dtype).to(dev)  # one projection: the convolution's rows and the steps
        self.x, self.steps = rows[..., :self.C], rows[..., self.C:]
        self.weight, self.bias = (r(self.C, W) / 2).to(dtype).to(dev), (r(self.C) / 4).to(dtype).to(dev)
        self.state = r(B, W - 1, self.C).to(dtype).to(dev)
        self.rates, self.skip, self.step_bias = -torch.exp(r(H)).to(dev), r(H).to(dev), (r(H) - 2).to(dev)
        self.memory = r(B, H, P, N).to(dev)

    def split(self, y):
        H, P, G, N = self.shape
        v, k, q = y.split([H * P, G * N, G * N], -1)
        return k.unflatten(-1, (G, N)), v.unflatten(-1, (H, P)), q.unflatten(-1, (G, N))

    def __call__(self, x, steps, state, memory, lengths=None):
        y, state = cuda_ops.cuda_short_conv(x, self.weight, self.bias, state, activation="silu", lengths=lengths)
        h, memory = cuda_ops.cuda_selective_scan(*self.split(y), steps, self.rates, memory, skip=self.skip,
                                                 step_bias=self.step_bias, softplus=True, lengths=lengths)
        return h, state, memory

    def step(self, x, steps, state, memory):
        """One token, both states in place."""
        y, _ = cuda_ops.cuda_short_conv_step(x, state, self.weight, self.bias, activation="silu", state_out=state)
        return cuda_ops.cuda_selective_step(*self.split(y), steps, self.rates, memory, skip=self.skip,
                                            step_bias=self.step_bias, softplus=True, memory_out=memory)[0]

    def check(self, hidden, memory, lengths=None):
        """Against the float64 definition.  An element of the convolution's output y is off by its own rounding, half
        a step of |y|, and by (W + 8) 2^-24 of the sum s of its magnitudes (silu's slope is below 1.1); |y| <= s.  A
        product of the scan holds three of them, or two in the memory: 3 (e + (W + 9) 2^-24) of the scan's magnitudes
        over s, on top of the scan's own bound."""
        x, w, b, st = oracle.to64(self.x, self.weight, self.bias, self.state)
        y, _ = oracle.short_conv(x, w, b, st, lengths, True)
        s, _ = oracle.short_conv(x.abs(), w.abs(), b.abs(), st.abs(), lengths, False)
        steps, rates, mem, skip, bias = oracle.to64(self.steps, self.rates, self.memory, self.skip, self.step_bias)
        ref, rmem = oracle.selective_scan(*self.split(y), steps, rates, mem, skip, bias, lengths, True)
        mag, mmag = oracle.selective_scan(*self.split(s * 1.1), steps, rates, mem.abs(), skip.abs(), bias, lengths, True)
        e, lossy = half(self.dtype) if self.dtype != torch.float32 else 0, self.dtype == torch.bfloat16
        T, N = self.x.shape[1], self.shape[3]
        most = 3.03 * (e + (self.weight.shape[1] + 9) * U) + (N + 160 + T / 8) * U
        for got, want, m, own in ((hidden, ref, mag, half(hidden.dtype) * 1.001), (memory, rmem, mmag, U)):
            bound = own * want.abs() + (most + (e if lossy else 0)) * m
            off = (got.double().cpu() - want).abs() / bound
            assert (off <= 1).all() or bound.min() == 0 and ((off <= 1) | off.isnan()).all(), f"{off.nan_to_num(99).max():.2f} of the bound"


DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", DTYPES)
def test_padded_prompt_then_single_tokens(dev, dtype):
    """Prompts of unequal lengths, then every sequence's own next tokens, in place: the definition over whole sequences."""
    B, T, more = 3, 90, 5
    a = Layer(dev, dtype, B, T + more, seed=1)
    n = torch.tensor([T, 1, 66], device=dev)
    h, state, memory = a(a.x[:, :T], a.steps[:, :T], a.state, a.memory, n)
    rows = torch.zeros(B, T + more, *a.shape[:2], dtype=dtype, device=dev)
    rows[:, :T] = h
    at = torch.arange(B, device=dev)
    for i in range(more):
        rows[at, n + i] = a.step(a.x[at, n + i], a.steps[at, n + i], state, memory)
    a.check(rows, memory, n + more)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths", [None, (150, 70)])
def test_training_pass(dev, dtype, lengths):
    """Through both operators at once: the gradients of the parts, chained by hand, to the bit."""
    a = Layer(dev, dtype, 2, 150, seed=2)
    n = None if lengths is None else torch.tensor(lengths, device=dev)
    names = ("x", "steps", "weight", "bias", "state", "memory", "rates", "skip", "step_bias")
    for k in names:
        setattr(a, k, getattr(a, k).detach().requires_grad_())
    h, state, memory = a(a.x, a.steps, a.state, a.memory, n)
    a.check(h.detach(), memory.detach(), n)
    ups = [torch.randn_like(t) for t in (h, state, memory)]
    got = dict(zip(names, torch.autograd.grad((h, state, memory), [getattr(a, k) for k in names], ups)))

    y, state = cuda_ops.cuda_short_conv(a.x, a.weight, a.bias, a.state, activation="silu", lengths=n)
    cut = y.detach().requires_grad_()
    h, memory = cuda_ops.cuda_selective_scan(*a.split(cut), a.steps, a.rates, a.memory, skip=a.skip,
                                             step_bias=a.step_bias, softplus=True, lengths=n)
    late = ("steps", "memory", "rates", "skip", "step_bias")
    dcut, *rest = torch.autograd.grad((h, memory), [cut] + [getattr(a, k) for k in late], (ups[0], ups[2]))
    first = torch.autograd.grad((y, state), [getattr(a, k) for k in names if k not in late], (dcut, ups[1]))
    want = dict(zip(late, rest)) | dict(zip((k for k in names if k not in late), first))
    for k in names:
        assert torch.equal(got[k], want[k]), k


def test_gradient_against_differences(dev):
    """Of a float32 layer, along random directions of each input: central differences of the float64 definition,
    whose own error (third derivatives times 1e-8) is far below the float32 sums' 1e-4 of the gradient's size."""
    a = Layer(dev, torch.float32, 1, 40, H=2, P=8, G=1, N=8, seed=3)
    names = ("x", "steps", "weight", "bias", "state", "memory", "rates", "skip", "step_bias")
    x64 = dict(zip(names, oracle.to64(*(getattr(a, k) for k in names))))
    for k in names:
        setattr(a, k, getattr(a, k).detach().requires_grad_())
    h, state, memory = a(a.x, a.steps, a.state, a.memory)
    g = torch.Generator().manual_seed(3)
    ups = [torch.randn(t.shape, generator=g) for t in (h, state, memory)]
    grads = torch.autograd.grad((h, state, memory), [getattr(a, k) for k in names], [u.to(dev) for u in ups])

    def loss(v):
        y, s = oracle.short_conv(v["x"], v["weight"], v["bias"], v["state"], None, True)
        h, m = oracle.selective_scan(*a.split(y), v["steps"], v["rates"], v["memory"], v["skip"], v["step_bias"], None, True)
        return sum((u * t).sum() for u, t in zip(ups, (h, s, m)))

    for k, grad in zip(names, grads):
        grad = grad.double().cpu()
        way = torch.randn(grad.shape, generator=g, dtype=torch.float64)
        diff = (loss({**x64, k: x64[k] + 1e-4 * way}) - loss({**x64, k: x64[k] - 1e-4 * way})) / 2e-4
        assert abs((grad * way).sum() - diff) <= 1e-4 * grad.norm() * way.norm(), k


def captured(fn):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fn()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fn()
    return graph, out


def test_captured_serving_step(dev):
    """The layer's single token with both states in place, replayed with other work between: to the bit the eager loop's."""
    a = Layer(dev, torch.bfloat16, 4, 8, seed=4)
    x, steps, state, memory = a.x[:, 0].clone(), a.steps[:, 0].clone(), a.state.clone(), a.memory.clone()
    graph, out = captured(lambda: a.step(x, steps, state, memory))
    state.copy_(a.state), memory.copy_(a.memory)
    s2, m2 = a.state.clone(), a.memory.clone()
    for t in range(8):
        x.copy_(a.x[:, t]), steps.copy_(a.steps[:, t])
        graph.replay()
        want = a.step(a.x[:, t], a.steps[:, t], s2, m2)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(state, s2) and torch.equal(memory, m2)
        torch.randn(999, 999, device=dev).sum().item()


def test_captured_prompts_and_gradients(dev):
    """Two graphs in turn, one of a prompt cut in time parts, one of a prompt with its gradients, each with its own
    workspace: every replay to the bit the eager results."""
    ops = torch.ops.grm_cuda
    a = Layer(dev, torch.bfloat16, 1, 2200, H=1, P=16, G=1, N=24, seed=5)
    b = Layer(dev, torch.bfloat16, 2, 300, seed=6)
    b.x, b.steps = b.x.contiguous(), b.steps.contiguous()
    up = torch.randn(2, 300, *b.shape[:2], device=dev).to(torch.bfloat16)

    def train():
        y, _ = ops.short_conv_forward(b.x, b.weight, b.bias, b.state, None, True)
        args = (*b.split(y), b.steps, b.rates)
        h, _, states = ops.selective_scan_forward(*args, b.memory, b.skip, b.step_bias, None, True, True)
        dk, dv, dq, *rest = ops.selective_scan_backward(up, None, *args, b.skip, b.step_bias, None, states, True)
        dy = torch.cat([t.flatten(2) for t in (dv, dk, dq)], -1)
        return (h, *rest, *ops.short_conv_backward(dy, None, b.x, b.weight, b.bias, b.state, None, True))

    fns = (lambda: a(a.x, a.steps, a.state, a.memory), train)
    graphs = [captured(f) for f in fns]
    for turn in range(3):
        for lay in (a, b):
            for t in (lay.x, lay.steps, lay.memory):
                t.copy_(torch.randn_like(t))
        want = [f() for f in fns]
        for g, outs in graphs:
            for o in outs:
                o.fill_(9)
        graphs[0][0].replay(), graphs[1][0].replay()
        torch.randn(999, 999, device=dev).sum().item()
        for (_, outs), ref in zip(graphs, want):
            for i, (o, r) in enumerate(zip(outs, ref)):
                assert torch.equal(o, r), (turn, i)


def test_two_streams_at_once(dev):
    """Forward and backward of two layers side by side on two streams, neither the default: each its own results."""
    lays = [Layer(dev, torch.bfloat16, 1, 2200, H=2, P=16, G=1, N=24, seed=s) for s in (7, 8)]

    def go(a):
        leaves = [t.detach().requires_grad_() for t in (a.x, a.steps, a.memory)]
        h, state, memory = a(leaves[0], leaves[1], a.state, leaves[2])
        return h, state, memory, *torch.autograd.grad((h, memory), leaves, (torch.ones_like(h), torch.ones_like(memory)))

    want = [go(a) for a in lays]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in lays]
    got = [[], []]
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = go(lays[i])
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for i, (x, y) in enumerate(zip(g, w)):
            assert torch.equal(x, y), i


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_at_any_offset(dev, dtype):
    """Slices that begin off every wide load's boundary, and rows of an odd width: the packed copies' results."""
    a = Layer(dev, dtype, 2, 100, H=2, P=24, G=1, N=40, seed=9)
    wide = torch.randn(2, 100, a.C + 5, device=dev).to(dtype)
    wide[..., 1:a.C + 1] = a.x
    h, state, memory = a(wide[..., 1:a.C + 1], a.steps, a.state, a.memory)
    want = a(a.x.contiguous(), a.steps.contiguous(), a.state, a.memory)
    assert torch.equal(h, want[0]) and torch.equal(state, want[1]) and torch.equal(memory, want[2])
    k, v, q = a.split(wide[..., 1:a.C + 1])
    args = (a.steps, a.rates, a.memory)
    more = dict(skip=a.skip, step_bias=a.step_bias, softplus=True)
    got = cuda_ops.cuda_selective_scan(k, v, q, *args, **more)
    want = cuda_ops.cuda_selective_scan(k.contiguous(), v.contiguous(), q.contiguous(), *args, **more)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_past_32_bits(dev):
    """More than 2^31 elements of x, and of the scan's values: the last tokens as a call of their own gives them."""
    T, cut = 1_100_100, 1_100_000
    a = Layer(dev, torch.bfloat16, 1, 100, H=32, P=64, G=1, N=16, seed=10)
    assert T * a.C > 2 ** 31 and T * 32 * 64 > 2 ** 31
    g = torch.Generator(device=dev).manual_seed(10)
    x = torch.empty(1, T, a.C, dtype=torch.bfloat16, device=dev).normal_(generator=g)
    steps = torch.empty(1, T, 32, dtype=torch.bfloat16, device=dev).normal_(generator=g)
    h, state, memory = a(x, steps, a.state, a.memory)
    _, s0, m0 = a(x[:, :cut], steps[:, :cut], a.state, a.memory)
    h1, s1, m1 = a(x[:, cut:], steps[:, cut:], s0, m0)
    assert torch.equal(state, s1)
    # Chunks begin elsewhere, so each result lies anywhere inside its own bound: half a step of bfloat16 of what is
    # summed, and in float32 as many roundings as the tokens that the decays remember bring (256 chunks and more).
    y, _ = cuda_ops.cuda_short_conv(x[:, cut:], a.weight, a.bias, s0, activation="silu")
    mag, mmag = cuda_ops.cuda_selective_scan(*a.split(y.abs().float()), steps[:, cut:].float(), a.rates, m0.abs(),
                                             skip=a.skip.abs(), step_bias=a.step_bias, softplus=True)
    assert ((memory - m1).abs() <= 2 * (16 + 160 + 4 * 256) * U * mmag).all()
    assert ((h[:, cut:].float() - h1.float()).abs() <= 2.1 * 2.0 ** -8 * (mag + h1.float().abs())).all()


def test_empty_batches(dev):
    """No sequences: empty results, and the parameters' gradients zeros."""
    a = Layer(dev, torch.bfloat16, 0, 20, seed=11)
    names = ("x", "steps", "weight", "bias", "state", "memory", "rates", "skip", "step_bias")
    for k in names:
        setattr(a, k, getattr(a, k).detach().requires_grad_())
    h, state, memory = a(a.x, a.steps, a.state, a.memory)
    assert h.shape == (0, 20, 4, 32) and state.shape == (0, 3, a.C) and memory.shape == (0, 4, 32, 32)
    grads = torch.autograd.grad((h, state, memory), [getattr(a, k) for k in names],
                                [torch.ones_like(t) for t in (h, state, memory)])
    for k, g in zip(names, grads):
        assert g.shape == getattr(a, k).shape and not g.any(), k
    with torch.no_grad():
        assert a.step(a.x[:, 0], a.steps[:, 0], a.state.clone(), a.memory.clone()).shape == (0, 4, 32)


def test_the_torch_forms_on_the_gpu(dev):
    """``enabled=False``: the PyTorch forms, float32 too, so both within the definition's bound."""
    a = Layer(dev, torch.float32, 2, 70, seed=12)
    off = dict(enabled=False, activation="silu")
    y, s = cuda_ops.cuda_short_conv(a.x, a.weight, a.bias, a.state, **off)
    h, m = cuda_ops.cuda_selective_scan(*a.split(y), a.steps, a.rates, a.memory, skip=a.skip, step_bias=a.step_bias,
                                        softplus=True, enabled=False)
    a.check(h, m)
    a.check(*a(a.x, a.steps, a.state, a.memory)[::2])


def test_no_second_derivatives(dev):
    """A gradient of a gradient is refused, not taken as zero."""
    a = Layer(dev, torch.float32, 1, 9, seed=13)
    a.x, a.steps = a.x.detach().requires_grad_(), a.steps.detach().requires_grad_()
    y, _ = cuda_ops.cuda_short_conv(a.x, a.weight, a.bias, a.state, activation="silu")
    (dx,) = torch.autograd.grad(y.square().sum(), a.x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dx.square().sum(), a.x)
    h, _ = cuda_ops.cuda_selective_scan(*a.split(y.detach()), a.steps, a.rates, a.memory)
    (ds,) = torch.autograd.grad(h.square().sum(), a.steps, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(ds.square().sum(), a.steps)
