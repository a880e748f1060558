"""The group norm on the GPU against its float64 definition.

Tolerances.  A group's sums have W terms: mean and variance are off by at most W 2^-24 of the magnitudes that are
summed, so a normalised value by (W + 16) 2^-24 of (|x| + |mean|) r, the mean's cancellation included; sigmoid
takes an exponential of z (off by |z| + 4 steps) and a reciprocal.  Gradients: the same of each term, W more for the two means;
the weights' sums over R rows R more.  Last, half a step of the output's type."""

import pytest
import torch

import delta_oracle as oracle
from rnn_with_grm_amd import cuda_ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]

# rows, groups, width, gate, center, silu, weight, bias
CASES = [
    (1, 1, 1, False, True, False, True, True), (3, 7, 45, False, True, True, True, True), (300, 16, 128, True, False, True, True, False),
    (5, 2, 4096, True, True, False, True, True), (1000, 1, 3, False, True, False, False, True), (65, 3, 600, True, True, True, True, True),
    (33, 300, 8, True, True, True, True, True), (7, 2, 1000, False, True, True, True, False), (9, 5, 33, True, False, True, False, False),
    (2, 1, 2048, False, False, True, True, True), (70, 1, 320, True, False, False, True, True), (0, 2, 16, True, True, True, True, True),
    (4100, 4, 64, True, False, True, True, False), (17, 64, 16, False, True, False, False, False),
]


def inputs(dev, R, G, W, gate, weight, bias, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    C = G * W
    x = (r(R, C + 8) + 0.5).to(dtype).to(dev)[:, 8:]
    return (x, (1 + 0.3 * r(C)).to(dtype).to(dev) if weight else None, r(C).to(dtype).to(dev) if bias else None,
            r(R, C + 16).to(dtype).to(dev)[:, :C] if gate else None), r(R, C).to(dtype).to(dev)


def near(got, ref, bound, what):
    got = got.detach().double().cpu()
    assert got.shape == ref.shape, what
    eps = torch.finfo(torch.float32 if got.dtype == torch.float64 else got.dtype).eps
    assert eps and torch.isfinite(got).all()
    if ref.numel():
        worst = ((got - ref).abs() / bound).max()
        assert worst <= 1, f"{what}: {worst:.2f} of the bound"


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,G,W,gate,center,silu,weight,bias", CASES)
def test_forward_and_gradients(dev, R, G, W, gate, center, silu, weight, bias, dtype):
    args, go = inputs(dev, R, G, W, gate, weight, bias, dtype)
    leaves = [None if t is None else t.detach().requires_grad_() for t in args]
    call = lambda x, w, b, z: cuda_ops.cuda_group_norm(x, G, w, b, z, activation="silu" if silu else None, center=center)  # noqa: E731
    out = call(*leaves)
    assert out.dtype == dtype and torch.equal(out, call(*args))
    ref = oracle.to64(*args, grad=True)
    want = oracle.group_norm(ref[0], G, *ref[1:], silu, center)
    h = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal
    x, w, b, z = (None if t is None else t.detach() for t in ref)
    xg = x.view(R, G, W)
    mean = xg.mean(-1, keepdim=True) if center else torch.zeros_like(xg[..., :1])
    r = 1 / torch.sqrt((xg - mean).square().mean(-1, keepdim=True) + 1e-5)
    n = ((xg - mean) * r).flatten(1)
    nmag = ((xg.abs() + mean.abs()) * r * (1 + ((xg - mean) * r).abs())).flatten(1)  # of n: its own terms, and the variance's of it
    wa, ba = (torch.ones_like(x[:1]) if w is None else w.abs()), (0 if b is None else b.abs())
    ymag, y = nmag * wa + ba, n * (1 if w is None else w) + (0 if b is None else b)
    steps = (W + 16) * U
    arg = y if z is None else z
    zmag = arg.abs() + 8 + (ymag if z is None else 0)
    amag = arg.abs() + (ymag if z is None else 0)
    bound = h * want.detach().abs() * 1.001 + tiny + (steps * 1.2 * (ymag + amag) * (zmag if silu else 1) if z is None else
                                                      steps * amag * (ymag + y.abs()) * (zmag if silu else 1))
    near(out, want.detach(), bound, "out")
    got = torch.autograd.grad(out, [t for t in leaves if t is not None], go)
    exp = torch.autograd.grad(want, [t for t in ref if t is not None], go.double().cpu())
    assert [t.dtype for t in got] == [t.dtype for t in leaves if t is not None]
    d = go.double().cpu().abs()
    slope = zmag if silu else torch.ones_like(d)
    dy = d * ((1.2 * slope * slope) if z is None else amag * slope) + tiny
    dn = (dy * wa).view(R, G, W)
    ng = nmag.view(R, G, W)
    dxm = (r * (dn + ng * (dn * ng).mean(-1, keepdim=True) + dn.mean(-1, keepdim=True)) * (1 + ng)).flatten(1)
    bounds = [3 * steps * dxm]
    if w is not None:
        bounds.append((3 * steps + R * U) * (dy * nmag).sum(0))
    if b is not None:
        bounds.append((3 * steps + R * U) * dy.sum(0))
    if z is not None:
        bounds.append(3 * steps * d * (ymag + y.abs()) * 1.2 * slope * slope)
    for name, a, e, m in zip([k for k, t in zip("xwbz", leaves) if t is not None], got, exp, bounds):
        near(a, e, h * e.abs() * 1.001 + m + 2 * tiny, name)


def test_shapes_weights_and_streams(dev):
    (x, w, b, z), _ = inputs(dev, 24, 4, 32, True, True, True, torch.bfloat16)
    want = cuda_ops.cuda_group_norm(x, 4, w, b, z, activation="silu")
    shaped = cuda_ops.cuda_group_norm(x.contiguous().view(2, 3, 4, 128), 4, w, b, z.contiguous().view(2, 3, 4, 128), activation="silu")
    assert shaped.shape == (2, 3, 4, 128) and torch.equal(shaped.view(24, 128), want)
    assert torch.equal(cuda_ops.cuda_group_norm(x[0], 4, w, b, z[0], activation="silu"), want[0])
    assert torch.equal(cuda_ops.cuda_group_norm(x, 4, w.float(), b.float(), z, activation="silu"), want)
    turned = x.t().contiguous().t()
    assert torch.equal(cuda_ops.cuda_group_norm(turned, 4, w, b, z, activation="silu"), want)
    leaf = x[:1].clone().requires_grad_()
    out = cuda_ops.cuda_group_norm(leaf.expand(24, -1), 4, w, b, z)
    (g,) = torch.autograd.grad(out.float().sum(), leaf)
    assert g.shape == leaf.shape
    wl = w.float().requires_grad_()
    first = torch.autograd.grad(cuda_ops.cuda_group_norm(x, 4, wl, None, z).float().square().sum(), wl)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = torch.autograd.grad(cuda_ops.cuda_group_norm(x, 4, wl, None, z).float().square().sum(), wl)[0]
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, again)


def test_odd_values_stay_in_their_group(dev):
    (x, w, b, z), _ = inputs(dev, 6, 4, 40, True, True, True, torch.float32)
    want = cuda_ops.cuda_group_norm(x, 4, w, b, z, activation="silu")
    y = x.clone()
    y[2, 50] = float("inf")
    y[3, 0] = float("nan")
    got = cuda_ops.cuda_group_norm(y, 4, w, b, z, activation="silu")
    mask = torch.zeros_like(got, dtype=torch.bool)
    mask[2, 40:80], mask[3, :40] = True, True
    assert not torch.isfinite(got[mask]).all() and torch.equal(got[~mask], want[~mask])
    same = torch.full((2, 80), 3.0, device=dev)  # no variance: eps alone divides
    assert not cuda_ops.cuda_group_norm(same, 2).any()


def test_captured_with_its_gradients(dev):
    (x, w, b, z), go = inputs(dev, 200, 4, 64, True, True, True, torch.bfloat16)
    x, z = x.contiguous(), z.contiguous()

    def work():  # leaves of its own: no graph of them lives outside
        leaves = [t.detach().requires_grad_() for t in (x, w, b, z)]
        out = cuda_ops.cuda_group_norm(leaves[0], 4, *leaves[1:], activation="silu")
        return (out.detach(), *torch.autograd.grad(out, leaves, go))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work()
    for i in range(4):
        x.copy_(torch.randn_like(x.float()))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, e) for a, e in zip(got, work()))


def test_refusals(dev):
    x = torch.zeros(3, 12, device=dev)
    for kw, match in [(dict(groups=5), "multiple"), (dict(weight=x[0, :4]), "weight"), (dict(weight=x[0].half()), "weight"),
                      (dict(weight=x[0], bias=x[0].bfloat16()), "bias"), (dict(gate=x[:2]), "gate"), (dict(gate=x.half()), "gate"),
                      (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(activation="relu"), "activation"),
                      (dict(weight=x[0].cpu()), "must be on")]:
        kw = dict(dict(groups=3), **kw)
        with pytest.raises(ValueError, match=match):
            cuda_ops.cuda_group_norm(x, kw.pop("groups"), **kw)
    with pytest.raises(ValueError, match="4096"):
        cuda_ops.cuda_group_norm(torch.zeros(1, 4097, device=dev), 1)
    with pytest.raises(ValueError, match="float32, float16"):
        cuda_ops.cuda_group_norm(x.double(), 3)
