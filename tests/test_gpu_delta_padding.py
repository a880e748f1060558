"""The delta rule behind the lengths of a padded batch, also where live tokens, states or gradients hold values that are no
numbers.  What is compared here has to be equal: zeros, states that nothing moves, and rows that nothing reaches."""

import pytest
import torch

from rnn_with_grm_amd import cuda_ops

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
NAMES = ("keys", "values", "queries", "strengths", "log_decays", "memory")


def inputs(dev, B, T, H, P, G, N, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    unit = lambda *s: 0.99 * torch.nn.functional.normalize(r(*s), dim=-1)  # noqa: E731
    x = [unit(B, T, G, N).to(dtype), r(B, T, H, P).to(dtype), unit(B, T, G, N).to(dtype), torch.rand(B, T, H, generator=g).to(dtype),
         -0.05 * torch.rand(B, T, H, generator=g), r(B, H, P, N)]
    return dict(zip(NAMES, (t.to(dev) for t in x)))


def run(x, n):
    return cuda_ops.cuda_delta_scan(*(x[k] for k in NAMES), lengths=n)


# Where a bad value of sequence 0 goes, and what is NaN of it from its token on: a column of head 1, a row, head 1, or the group.
PLACES = [("values", (1, 5), "column"), ("queries", (0, 3), "row"), ("keys", (0, 3), "group"), ("strengths", (1,), "head"),
          ("log_decays", (1,), "head"), ("memory", (1, 5, 3), "column")]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,P,N,lengths,at", [(20, 40, 32, (10, 20), 5), (150, 40, 128, (100, 7), 77), (150, 37, 65, (100, 0), 70),
                                              (70, 64, 64, (65, 64), 64), (3000, 24, 48, (1500, 2990), 1400),
                                              (3000, 70, 48, (3000, 2990), 700)])
def test_rows_behind_a_length_are_zeros(dev, T, P, N, lengths, at, dtype):
    x = inputs(dev, 2, T, 2, P, 1, N, dtype, seed=T)
    n = torch.tensor(lengths, device=dev)
    hidden, memory = run(x, n)
    live = torch.arange(T, device=dev) < n[:, None]
    assert not hidden[~live].any()
    for bad in (float("inf"), float("nan")):
        for name, where, what in PLACES:
            y = dict(x, **{name: x[name].clone()})
            y[name][(0, *where) if name == "memory" else (0, at, *where)] = bad
            h, m = run(y, n)
            assert torch.equal(h[~live], torch.zeros_like(h[~live])), (name, bad)
            odd, gone = torch.zeros_like(h, dtype=torch.bool), torch.zeros_like(m, dtype=torch.bool)
            start = 0 if name == "memory" else at
            if what == "column":
                odd[0, start:, 1, 5], gone[0, 1, 5] = True, True
            elif what == "row":
                odd[0, at] = True
            elif what == "head":
                odd[0, start:, 1], gone[0, 1] = True, True
            else:
                odd[0, start:], gone[0] = True, True
            odd &= live[..., None, None]
            assert torch.equal(torch.isnan(h), odd) and torch.equal(torch.isnan(m), gone), (name, bad)
            assert torch.equal(h[~odd], hidden[~odd]) and torch.equal(m[~gone], memory[~gone]), (name, bad)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,P,N,lengths,at", [(20, 40, 32, (10, 20), 5), (150, 40, 128, (100, 7), 77), (150, 37, 65, (100, 0), 70),
                                              (3000, 24, 48, (1500, 2990), 1400), (3000, 70, 48, (2999, 2990), 700)])
def test_gradients_behind_a_length_are_zeros(dev, T, P, N, lengths, at, dtype):
    """Also where a live value, state or gradient is no number; the other sequence's gradients are what they were."""
    x = inputs(dev, 2, T, 2, P, 1, N, dtype, seed=T)
    n = torch.tensor(lengths, device=dev)
    live = torch.arange(T, device=dev) < n[:, None]
    g = torch.Generator().manual_seed(1)
    seeds = [torch.randn(2, T, 2, P, generator=g).to(dtype).to(dev), torch.randn(2, 2, P, N, generator=g).to(dev)]

    def gradients(x, seeds):
        leaves = [x[k].detach().requires_grad_() for k in NAMES]
        return torch.autograd.grad(cuda_ops.cuda_delta_scan(*leaves, lengths=n), leaves, seeds)

    want = gradients(x, seeds)
    for bad in (float("inf"), float("nan")):
        for name, where, _ in PLACES + [("hidden", (1, 5), ""), ("memory_out", (1, 5, 3), "")]:
            y, s = dict(x), list(seeds)
            if name in y:
                to = y[name] = y[name].clone()
            else:
                i = ("hidden", "memory_out").index(name)
                to = s[i] = s[i].clone()
            to[(0, *where) if to.shape == x["memory"].shape else (0, at, *where)] = bad
            for k, a, b in zip(NAMES, gradients(y, s), want):
                if k != "memory":
                    assert torch.equal(a[~live], torch.zeros_like(a[~live])), (name, bad, k)
                assert torch.equal(a[1], b[1]), (name, bad, k)


@pytest.mark.parametrize("T", [100, 3000])
def test_a_state_that_no_token_moves(dev, T):
    """An empty sequence hands its state on as it is, in time parts too: infinities, NaN, the largest and the smallest numbers."""
    x = inputs(dev, 3, T, 1, 40, 1, 48, torch.bfloat16, seed=3)
    odd = torch.tensor([float("inf"), float("-inf"), float("nan"), 3.4028235e38, 1e-38, 1e-45, 1.0000001], device=dev)
    x["memory"][0, 0, ::6, 3] = odd
    x["memory"][2, 0, 3] = odd[3]
    n = torch.tensor([0, T // 2, -4], device=dev)
    hidden, memory = run(x, n)
    assert not hidden[0].any() and not hidden[2].any()
    for b in (0, 2):
        assert torch.equal(memory[b].view(torch.int32), x["memory"][b].view(torch.int32))
    assert torch.isfinite(memory[1]).all()
    # its gradient likewise
    leaves = [x[k].detach().requires_grad_() for k in NAMES]
    seed = torch.ones_like(memory)
    seed[0, 0, ::6, 3] = odd
    grads = torch.autograd.grad(cuda_ops.cuda_delta_scan(*leaves, lengths=n)[1], leaves, seed)
    for b in (0, 2):
        assert torch.equal(grads[5][b].view(torch.int32), seed[b].view(torch.int32))
        assert not any(t[b].any() for t in grads[:5])
