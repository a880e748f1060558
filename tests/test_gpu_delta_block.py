"""The delta rule as a block uses it: a short convolution in front, normalised keys, the norm with its gate behind;
prompts continued token by token, gradients through all of it, long sequences of few heads.

Tolerances.  A chain of T tokens with keys of at most unit length is off by 8 sqrt(T + 64) 2^-24 of its largest value (the
handful of float32 roundings of a token is not enlarged by later ones); the norm takes rows to unit scale, and rows here are seldom shorter than
a quarter of the usual length: four times that, in the root of the squares' sum.  bfloat16 rows are rounded at six places (convolution,
keys, queries, hidden rows, norm, and the convolution's state); two ways to the same row may round to neighbours,
one step each: 6 x 2^-7 of the rows, at most twice that behind the norm."""

import math

import pytest
import torch

import delta_oracle as oracle
from rnn_with_grm_amd import cuda_ops

pytestmark = pytest.mark.gpu
H, G, P, N, W = 4, 2, 32, 64, 4
C = H * P + 2 * G * N


def weights(dev, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    w = dict(conv=r(C, W) / 2, conv_bias=r(C) / 2, norm=1 + 0.1 * r(H * P))
    return {k: v.to(dtype).to(dev) for k, v in w.items()}


def block(w, x, beta, decay, gate, conv_state, memory, lengths=None):
    """One block over x [B, T, C]; T may be one."""
    rows, conv_state = cuda_ops.cuda_short_conv(x, w["conv"], w["conv_bias"], conv_state, activation="silu", lengths=lengths)
    v, k, q = rows.split((H * P, G * N, G * N), -1)
    k, q = (torch.nn.functional.normalize(t.unflatten(-1, (G, N)).float(), dim=-1).to(x.dtype) for t in (k, q))
    h, memory = cuda_ops.cuda_delta_scan(k, v.unflatten(-1, (H, P)), q, beta, decay, memory, lengths=lengths)
    y = cuda_ops.cuda_group_norm(h.flatten(-2), H, w["norm"], None, gate, activation="silu", center=False)
    return y, conv_state, memory


def token(w, x, beta, decay, gate, conv_state, memory):
    """One token, states moved in place."""
    rows, _ = cuda_ops.cuda_short_conv_step(x, conv_state, w["conv"], w["conv_bias"], activation="silu", state_out=conv_state)
    v, k, q = rows.split((H * P, G * N, G * N), -1)
    k, q = (torch.nn.functional.normalize(t.unflatten(-1, (G, N)).float(), dim=-1).to(x.dtype) for t in (k, q))
    h, _ = cuda_ops.cuda_delta_step(k, v.unflatten(-1, (H, P)), q, beta, decay, memory, memory_out=memory)
    return cuda_ops.cuda_group_norm(h.flatten(-2), H, w["norm"], None, gate, activation="silu", center=False)


def inputs(dev, B, T, dtype, seed=1):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return [t.to(dev) for t in (r(B, T, C).to(dtype), torch.sigmoid(r(B, T, H)).to(dtype), -torch.exp(r(B, T, H) - 2), r(B, T, H * P).to(dtype))]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_padded_prompt_goes_on_token_by_token(dev, dtype):
    B, T, more = 3, 150, 5
    w = weights(dev, dtype)
    x, beta, decay, gate = inputs(dev, B, T + more, dtype)
    n = torch.tensor([T, 70, 1], device=dev)
    y, conv, memory = block(w, x[:, :T], beta[:, :T], decay[:, :T], gate[:, :T], None, None, n)
    assert not y[1, 70:].any() and not y[2, 1:].any()
    steps = []
    for t in range(more):
        at = n + t
        pick = lambda z: z[torch.arange(B, device=dev), at]  # noqa: E731
        steps.append(token(w, pick(x), pick(beta), pick(decay), pick(gate), conv, memory))
    for b in range(B):
        end = int(n[b]) + more
        whole, _, last = block(w, x[b:b + 1, :end], beta[b:b + 1, :end], decay[b:b + 1, :end], gate[b:b + 1, :end], None, None)
        got = torch.cat([y[b, :end - more], torch.stack([s[b] for s in steps])]).double()
        want = whole[0].double()
        chain = 8 * math.sqrt(T + 64) * 2.0 ** -24
        bound = 4 * chain if dtype == torch.float32 else 12 * torch.finfo(dtype).eps
        assert (got - want).norm() <= bound * want.norm()
        bound = chain if dtype == torch.float32 else 6 * torch.finfo(dtype).eps
        assert (memory[b].double() - last[0].double()).norm() <= bound * last.double().norm()



def test_gradients_through_the_block(dev):
    """Float32: against the PyTorch forms of the three parts in float64."""
    w = weights(dev, torch.float32)
    args = inputs(dev, 2, 90, torch.float32)
    leaves = [t.requires_grad_() for t in args] + [t.requires_grad_() for t in w.values()]
    out = block(dict(zip(w, leaves[4:])), *leaves[:4], None, None)
    pick = [torch.randn_like(o) for o in (out[0], out[2])]
    got = torch.autograd.grad((out[0], out[2]), leaves, pick)
    ref = [t.detach().double().cpu().requires_grad_() for t in leaves]
    exp = block(dict(zip(w, ref[4:])), *ref[:4], None, None)
    want = torch.autograd.grad((exp[0], exp[2]), ref, [t.double().cpu() for t in pick])
    for a, b in zip(got, want):
        # four chains of sqrt(90 + 64) roundings, P N values a number at most, unit scale by the norm (sixteenfold)
        assert (a.double().cpu() - b).norm() <= 4 * 8 * math.sqrt(154) * 16 * 2.0 ** -24 * b.norm()


@pytest.mark.parametrize("dtype,P1,N1", [(torch.bfloat16, 40, 128), (torch.float32, 40, 64), (torch.bfloat16, 70, 90),
                                         (torch.float16, 130, 30), (torch.float32, 5, 7)])
def test_long_sequences_of_few_heads(dev, dtype, P1, N1):
    """In time parts, with gradients: whole and odd widths, odd numbers of column tiles."""
    g = torch.Generator().manual_seed(4)
    T = 3000
    unit = lambda: 0.99 * torch.nn.functional.normalize(torch.randn(1, T, 1, N1, generator=g), dim=-1)  # noqa: E731
    x = [unit().to(dtype).to(dev), torch.randn(1, T, 1, P1, generator=g).to(dtype).to(dev), unit().to(dtype).to(dev),
         torch.rand(1, T, 1, generator=g).to(dtype).to(dev), (-0.02 * torch.rand(1, T, 1, generator=g)).to(dev),
         torch.randn(1, 1, P1, N1, generator=g).to(dev)]
    leaves = [t.requires_grad_() for t in x]
    out = cuda_ops.cuda_delta_scan(*leaves)
    w = [torch.randn(o.shape, generator=g).to(o.dtype).to(dev) for o in out]
    got = torch.autograd.grad(out, leaves, w)
    ref = oracle.to64(*x, grad=True)
    exp = oracle.delta_scan(*ref, None)
    want = torch.autograd.grad(exp, ref, [t.double().cpu() for t in w])
    chain = 8 * math.sqrt(T + 64) * 2.0 ** -24
    for a, b in zip((*out, *got), (*exp, *want)):
        a, b = a.detach().double().cpu(), b.detach()
        # rounded once to 16 bits, from products of operands held to 2^-16 (no more than 2^-14 of the rows); a sum over P N numbers
        # of a token adds at most its own length
        bound = 4 * chain * (math.sqrt(P1 * N1) if a.shape == x[4].shape else 1)
        bound += 0 if dtype == torch.float32 else 2.0 ** -14 + torch.finfo(dtype).eps / 2
        assert (a - b).norm() <= bound * b.norm()


@pytest.mark.parametrize("T", [200, 3000])
def test_captured_gradients(dev, T):
    """Forward and backward of the delta rule in a graph, with leaves of its own, replayed between eager work; in time parts too."""
    x, beta, decay, _ = inputs(dev, 2, T, torch.bfloat16)
    rows = x.clone()
    seed = torch.randn(2, T, H, P, device=dev).bfloat16()

    def work():
        v, k, q = rows.split((H * P, G * N, G * N), -1)
        k, q = (torch.nn.functional.normalize(t.unflatten(-1, (G, N)).float(), dim=-1).bfloat16() for t in (k, q))
        leaves = [t.detach().requires_grad_() for t in (k, v.unflatten(-1, (H, P)), q, beta, decay)]
        h, m = cuda_ops.cuda_delta_scan(*leaves)
        return (h.detach(), m.detach(), *torch.autograd.grad((h, m), leaves, (seed, torch.ones_like(m))))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work()
    for i in range(4):
        rows.copy_(torch.randn_like(rows.float()))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, work()))
