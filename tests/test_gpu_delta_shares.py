"""Gradients of the delta rule where a workgroup takes several heads of a group, one after the other, and where long
sequences of several heads are walked in time parts beside padding.

The definition here is plain PyTorch in float64, token by token for the whole batch.  Tolerances: keys have at most unit length and
strengths lie in [0, 1], so no error made at a token grows, and those of T tokens (a chunk's 64 beside them) add up like the square
root: 8 sqrt(T + 64) 2^-24 of the largest value, 2^-14 more where operands are held to 2^-16 for 16-bit results.  Gradients pass four
such chains; a number of a token that is summed over a head's values and keys adds sqrt(P N); keys' and queries' gradients
are sums over the heads of a group, whose errors are independent: the square root of their number.  Then half a step of the type."""

import math

import pytest
import torch

from rnn_with_grm_amd import capi, cuda_ops

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
NAMES = ("keys", "values", "queries", "strengths", "log_decays", "memory")


def definition(k, v, q, b, g, M, n):
    T, H, G = v.size(1), v.size(2), k.size(2)
    k, q = (t.repeat_interleave(H // G, 2) for t in (k, q))
    rows = []
    for t in range(T):
        live = (t < n).double()[:, None]
        M = torch.exp(g[:, t] * live)[..., None, None] * M
        u = (b[:, t] * live)[..., None] * (v[:, t] - (M * k[:, t, :, None]).sum(-1))
        M = M + u[..., None] * k[:, t, :, None]
        rows.append((M * q[:, t, :, None]).sum(-1) * live[..., None])
    return torch.stack(rows, 1), M


def check(dev, B, T, H, P, G, N, lengths, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    unit = lambda: 0.99 * torch.nn.functional.normalize(r(B, T, G, N), dim=-1)  # noqa: E731
    x = [unit(), r(B, T, H, P), unit(), torch.rand(B, T, H, generator=g)]
    x = [t.to(dtype) for t in x] + [-0.05 * torch.rand(B, T, H, generator=g), r(B, H, P, N)]
    seeds = [r(B, T, H, P).to(dtype), r(B, H, P, N)]
    n = torch.full((B,), T) if lengths is None else lengths
    leaves = [t.to(dev).requires_grad_() for t in x]
    out = cuda_ops.cuda_delta_scan(*leaves, lengths=None if lengths is None else n.to(dev))
    got = torch.autograd.grad(out, leaves, [s.to(dev) for s in seeds])
    ref = [t.to(dev).double().requires_grad_() for t in x]
    exp = definition(*ref, n.to(dev))
    want = torch.autograd.grad(exp, ref, [s.to(dev).double() for s in seeds])
    for name, a, e in zip(("hidden", "memory_out", *NAMES), (*out, *got), (*exp, *want)):
        a, e = a.detach().double(), e.detach()
        kind = torch.float32 if name in ("memory_out", "log_decays", "memory") else dtype
        rel = 8 * math.sqrt(T + 64) * 2.0 ** -24 + (2.0 ** -14 if kind != torch.float32 else 0)
        if name not in ("hidden", "memory_out"):
            rel *= 4 * (math.sqrt(P * N) if name in ("strengths", "log_decays") else math.sqrt(H // G) if name in ("keys", "queries") else 1)
        bound = torch.finfo(kind).eps / 2 * 1.001 * e.abs() + rel * e.abs().max() + torch.finfo(kind).smallest_normal
        assert torch.isfinite(a).all() and ((a - e).abs() <= bound).all(), (name, ((a - e).abs() / bound).max())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,H,P,G,N,padded", [
    (64, 130, 5, 16, 1, 24, False),   # 192 chunks of a group: three shares of two, two and one head
    (64, 130, 5, 40, 1, 72, True),
    (100, 130, 14, 8, 2, 16, True),   # 600: seven heads of a group in one workgroup
    (180, 129, 3, 70, 1, 128, True)])
def test_several_heads_of_a_workgroup(dev, B, T, H, P, G, N, padded, dtype):
    lengths = torch.randint(0, T + 1, (B,), generator=torch.Generator().manual_seed(2)) if padded else None
    check(dev, B, T, H, P, G, N, lengths, dtype, B + N)


# 16 x 32 fragments of the triangular matrices' parts and a chunk's scalars, of every chunk: what a walk in one part needs.
def one_part(B, T, H, dtype):
    parts = 3 + (3 if dtype == torch.float32 else 2)
    return B * H * ((T + 63) // 64) * (parts * 6 * 512 * 2 + 208 * 4)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,P,G,N", [(2, 24, 2, 40), (3, 70, 1, 64)])
@pytest.mark.parametrize("lengths", [(0, 1500, 3000), (70, 2990, 704), (2000, 1, 64)])
def test_time_parts_of_several_heads_and_lengths(dev, H, P, G, N, lengths, dtype):
    B, T = 3, 3000
    code = {torch.float32: capi.F32, torch.float16: capi.F16, torch.bfloat16: capi.BF16}[dtype]
    assert capi.load().grm_hip_delta_scan_workspace(B, T, H, P, N, code) > one_part(B, T, H, dtype) + 16
    check(dev, B, T, H, P, G, N, torch.tensor(lengths), dtype, sum(lengths))
