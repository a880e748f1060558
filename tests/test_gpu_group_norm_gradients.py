"""The group norm's gradients against the formula in float64, with bounds that a dropped term exceeds, and what an infinity or a
NaN reaches.

Bounds.  Let d be the depth of a group's sums: the registers of a lane one after the other and then a tree over the lanes.  Of
dx = r (dn - n mean(dn n) - mean(dn)) no term is longer than |dn| (the norm over the group: |n| is at most sqrt(W), so
|n mean(dn n)| <= |dn|, and a mean's part of a vector is no longer than the vector).  n is off by (d + 8) 2^-24 of itself and of
the mean's rest, activations by their argument's error times a slope of at most 1.1 (silu' of it at most 0.5) and (4 + |z|) steps
of their own, z below 8 here; a mean by d steps of |dn|.  Three terms, their operands' errors and the products': 8 (d + 16) 2^-24 of
r |dn|, times the largest weight where it passes one, as n's error comes back through the activation."""

import pytest
import torch

import delta_oracle as oracle
from rnn_with_grm_amd import cuda_ops

pytestmark = pytest.mark.gpu


def depth(W):
    lanes = 1
    while lanes < 64 and lanes * 8 < W:
        lanes *= 2
    return max(8, -(-W // lanes)) + lanes.bit_length() - 1


@pytest.mark.parametrize("R,G,W,gate,center,silu", [
    (7, 2, 1000, False, True, True), (2, 1, 2048, False, False, True), (3, 7, 45, False, True, True), (5, 2, 4096, False, True, True),
    (33, 300, 8, False, True, True), (9, 4, 128, True, True, True), (16, 3, 600, True, False, True), (6, 5, 33, False, False, False),
    (40, 2, 320, True, True, False)])
def test_gradient_of_rows(dev, R, G, W, gate, center, silu):
    g = torch.Generator().manual_seed(W)
    r = lambda *s: torch.randn(*s, generator=g).clamp(-4, 4)  # noqa: E731
    x, z, d = r(R, G * W) + 0.5, r(R, G * W), r(R, G * W)
    w, b = 1 + 0.3 * r(G * W), 0.5 * r(G * W)
    leaf, gleaf = x.to(dev).requires_grad_(), z.to(dev).requires_grad_()
    out = cuda_ops.cuda_group_norm(leaf, G, w.to(dev), b.to(dev), gleaf if gate else None, activation="silu" if silu else None, center=center)
    got = torch.autograd.grad(out, (leaf, gleaf) if gate else (leaf,), d.to(dev))

    # The formula in float64, term by term.
    x, z, d, w, b = (t.double() for t in (x, z, d, w, b))
    xg = x.view(R, G, W)
    c = xg - xg.mean(-1, keepdim=True) if center else xg
    rr = 1 / torch.sqrt(c.square().mean(-1, keepdim=True) + 1e-5)
    n = c * rr
    y = n.flatten(1) * w + b
    u = z if gate else y
    sg = 1 / (1 + torch.exp(-u))
    act, slope = (u * sg, sg * (1 + u * (1 - sg))) if silu else (u, torch.ones_like(u))
    dn = ((d * act if gate else d * slope) * w).view(R, G, W)
    across, along = n * (dn * n).mean(-1, keepdim=True), dn.mean(-1, keepdim=True) if center else torch.zeros_like(rr)
    want = rr * (dn - across - along)
    ref = x.clone().requires_grad_()  # (and the definition's own gradient is the formula's)
    loss = oracle.group_norm(ref, G, w, b, z if gate else None, silu, center)
    torch.testing.assert_close(torch.autograd.grad(loss, ref, d)[0].view(R, G, W), want, rtol=1e-9, atol=1e-9)

    wmax = max(1.0, float(w.abs().max()))
    bound = 8 * (depth(W) + 16) * 2.0 ** -24 * wmax * (rr * dn.norm(dim=-1, keepdim=True)).squeeze(-1)
    off = lambda t: (t - want).norm(dim=-1) / bound  # noqa: E731
    assert off(got[0].double().cpu().view(R, G, W)).max() <= 1
    # Without either mean most groups would be far off.
    assert off(want + rr * across).median() > 10
    if center:
        assert off(want + rr * along).median() > 10
    if gate:
        # dgate = dout y act'(gate), an element at a time: y's error (d + 8 steps of |n w| and as much of the mean's rest), the slope's
        e = (got[1].double().cpu() - d * y * slope).abs()
        assert (e <= (2 * depth(W) + 32) * 2.0 ** -24 * d.abs() * (w.abs() * (n.flatten(1).abs() + 1) + b.abs()) * 1.1).all()


@pytest.mark.parametrize("center", [True, False])
@pytest.mark.parametrize("W", [40, 36, 600])
def test_what_a_value_that_is_no_number_reaches(dev, W, center):
    """Each element of its group as the definition has it, and no other group; of a row's gradient likewise."""
    g = torch.Generator().manual_seed(W)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x, z, w, b = r(6, 4 * W), r(6, 4 * W), r(4 * W), r(4 * W)
    call = lambda t: cuda_ops.cuda_group_norm(t.to(dev), 4, w.to(dev), b.to(dev), z.to(dev), activation="silu", center=center).cpu()  # noqa: E731
    clean = call(x)
    for bad in (float("inf"), float("-inf"), float("nan")):
        y = x.clone()
        y[2, W + 5] = bad
        got, want = call(y), oracle.group_norm(y.double(), 4, w.double(), b.double(), z.double(), True, center)
        mask = torch.zeros_like(got, dtype=torch.bool)
        mask[2, W:2 * W] = True
        assert torch.equal(got[~mask], clean[~mask])
        nan = torch.isnan(want)
        assert nan[mask].any() and torch.equal(torch.isnan(got), nan)
        if center or bad != bad:
            assert nan[mask].all()
        else:  # n is zero beside an infinity, so this is the bias by the gate
            torch.testing.assert_close(got[mask & ~nan].double(), want[mask & ~nan], rtol=1e-6, atol=1e-7)

    leaves = [t.to(dev).requires_grad_() for t in (x, w, b, z)]

    def gradients(d):
        out = cuda_ops.cuda_group_norm(leaves[0], 4, *leaves[1:], activation="silu", center=center)
        return [t.cpu() for t in torch.autograd.grad(out, leaves, d.to(dev))]

    d = r(6, 4 * W)
    want = gradients(d)
    d[3, 2 * W + 1] = float("nan")
    for name, a, e in zip("xwbz", gradients(d), want):
        mask = torch.zeros_like(a, dtype=torch.bool)
        if name == "x":
            mask[3, 2 * W:3 * W] = True
        else:
            mask[(3, 2 * W + 1) if a.ndim == 2 else 2 * W + 1] = True
        assert torch.equal(torch.isnan(a), mask) and torch.equal(a[~mask], e[~mask]), name
