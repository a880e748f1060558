"""Gradients of the selective scan where a workgroup walks several heads and value tiles: batches of many blocks, whose
groups' heads are shared by few workgroups or by none (256 workgroups and more).  Against the float64 definition, the
whole batch a token at a time; bounds as in test_gpu_selective_bwd, with what bfloat16 inputs lose in two parts of 8 bits."""

import pytest
import torch

import selective_oracle as oracle
from test_gpu_selective_bwd import magnitudes
from test_gpu_selective_scan import DTYPES, NAMES, inputs, near, run

pytestmark = pytest.mark.gpu
PARTS = 2.0 ** -16 * 1.01


def batched(keys, values, queries, steps, rates, memory, skip, step_bias, lengths, softplus):
    """oracle.selective_scan over all sequences at once."""
    B, T, H, P = values.shape
    G, N = keys.shape[2:]
    n = torch.tensor(oracle.lengths_of(lengths, B, T))
    M = torch.zeros(B, H, P, N, dtype=torch.float64) if memory is None else memory
    rows = []
    for t in range(T):
        live = t < n
        d = steps[:, t] if step_bias is None else steps[:, t] + step_bias
        d = torch.logaddexp(d, torch.zeros_like(d)) if softplus else d
        k, q = (v[:, t].repeat_interleave(H // G, 1) for v in (keys, queries))
        rate = rates if rates.ndim == 1 else rates[:, t]
        new = torch.exp(d * rate)[..., None, None] * M + (d[..., None] * values[:, t])[..., None] * k[:, :, None]
        M = torch.where(live[:, None, None, None], new, M)
        h = (M * q[:, :, None]).sum(-1)
        h = h if skip is None else h + skip[:, None] * values[:, t]
        rows.append(torch.where(live[:, None, None], h, 0.0))
    return (torch.stack(rows, 1) if rows else 1.0 * values), M


def test_the_batched_definition():
    g = torch.Generator().manual_seed(0)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    x = (r(3, 6, 2, 5), r(3, 6, 4, 3), r(3, 6, 2, 5), r(3, 6, 4), -torch.exp(r(4)), r(3, 4, 3, 5), r(4), r(4))
    n = torch.tensor([6, 0, 4])
    for a, b in zip(batched(*x, n, True), oracle.selective_scan(*x, n, True)):
        torch.testing.assert_close(a, b, rtol=1e-13, atol=1e-13)


CASES = [
    # B, T, H, P, G, N, ragged       (head, value tile) pairs of a group / workgroups that share them, bf16
    (256, 5, 6, 80, 1, 24, False),  # 12 / 1: one workgroup walks all heads and both tiles of their values
    (100, 9, 5, 16, 1, 64, False),  # 5 / 3: unequal shares
    (64, 130, 6, 80, 1, 40, True),  # 12 / 2, two blocks, some of them behind the length
    (130, 3, 6, 64, 2, 128, True),  # 3 / 1: two groups
    (300, 2, 3, 33, 1, 7, False),   # 3 / 1, rows of odd widths
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,H,P,G,N,ragged", CASES)
def test_gradients(dev, monkeypatch, B, T, H, P, G, N, ragged, dtype):
    monkeypatch.setattr(oracle, "selective_scan", batched)
    x = inputs(dev, B, T, H, P, G, N, dtype, seed=B + T)
    g = torch.Generator().manual_seed(B)
    n = torch.randint(-1, T + 2, (B,), generator=g).to(dev) if ragged else None
    dead = torch.zeros(B, T, dtype=torch.bool, device=dev)
    if ragged:
        dead = torch.arange(T, device=dev) >= n.clamp(0, T)[:, None]
        for k in ("keys", "values", "queries"):
            x[k] = x[k].masked_fill(dead[..., None, None], float("nan"))
    leaves = {k: x[k].detach().requires_grad_() for k in NAMES}
    outs = run(leaves, n)
    dy, dm = torch.randn(outs[0].shape, generator=g).to(dtype), torch.randn(outs[1].shape, generator=g)
    got = torch.autograd.grad(outs, [leaves[k] for k in NAMES], [dy.to(dev), dm.to(dev)])
    # (zeros in the place of NaN: 0 x NaN in the definition's own gradients)
    x64 = dict(zip(NAMES, (t.nan_to_num().requires_grad_() for t in oracle.to64(*(x[k] for k in NAMES)))))
    ref = batched(*(x64[k] for k in NAMES), n, True)
    want = torch.autograd.grad(ref, [x64[k] for k in NAMES], (dy.double(), dm.double()))
    mags = magnitudes(x64, n, True, dy.double(), dm.double())
    steps = N + P + 256 + T / 8 + 64 + B / 8  # (`rates`, `skip` and `step_bias` sum over the batch, too)
    for k, a, b in zip(NAMES, got, want):
        lossy = dtype == torch.bfloat16 and k in ("keys", "values", "queries")
        try:
            near(a, b, mags[k], a.dtype, PARTS if lossy else 0, steps)
        except AssertionError as e:
            raise AssertionError(f"gradient of {k}: {e}") from None
    for a in (outs[0], *got[:4]):
        assert (a[dead] == 0).all()
