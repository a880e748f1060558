"""The gated delta rule on the GPU against its float64 definition.

Tolerances.  Keys here have at most unit length and strengths lie in [0, 1], so a token's transition has no
norm above one: an error made at a token is not enlarged by the ones behind it, and those of T tokens, made
independently, add up like the square root of T.  At each a handful of float32 roundings is made of quantities no larger
than the largest that occur (a chunk's 64 tokens count as such in its sums): results are off by at most
8 sqrt(T + 64) 2^-24 of the largest value of their head.  16-bit outputs come from products whose operands are held to 2^-16
(half a step of either part: 2^-17, over sqrt(128) terms no more than 2^-14 of the largest), and are rounded
once, half a step of the value.  Gradients pass four such chains (forward, adjoint, and the products of both): four times
that; what is summed over a head's values and keys for one number of a token adds at most the sum's own length,
sqrt(P N) roundings."""

import math

import pytest
import torch

import delta_oracle as oracle
from rnn_with_grm_amd import cuda_ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
NAMES = oracle.NAMES


def half(dtype):
    return torch.finfo(dtype).eps / 2


def inputs(dev, B, T, H, P, G, N, dtype, seed, sdtype=None, ddtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    unit = lambda *s: 0.99 * torch.nn.functional.normalize(r(*s), dim=-1)  # noqa: E731  (at most one after rounding)
    return dict(keys=unit(B, T, G, N).to(dtype).to(dev), values=r(B, T, H * P + 8).to(dtype).to(dev)[..., 8:].unflatten(-1, (H, P)),
                queries=unit(B, T, G, N).to(dtype).to(dev), strengths=torch.rand(B, T, H, generator=g).to(sdtype or dtype).to(dev),
                log_decays=(-torch.exp(r(B, T, H) - 2)).to(ddtype).to(dev), memory=r(B, H, P, N).to(dev))


def run(x, lengths=None):
    return cuda_ops.cuda_delta_scan(*(x[k] for k in NAMES), lengths=lengths)


def near(got, ref, dtype, rel, what):
    got, ref = got.detach().double().cpu(), ref.detach()
    assert got.shape == ref.shape and torch.isfinite(got).all(), what
    if not ref.numel():
        return
    bound = half(dtype) * ref.abs() * 1.001 + rel * ref.abs().max() + torch.finfo(dtype).smallest_normal
    worst = ((got - ref).abs() / bound).max()
    assert worst <= 1, f"{what}: {worst:.2f} of the bound"


def tol(T, dtype):
    return 8 * math.sqrt(T + 64) * U + (2.0 ** -14 if dtype != torch.float32 else 0)


CASES = [
    # B, T, H, P, G, N, lengths
    (2, 1, 2, 64, 1, 64, None), (1, 2, 4, 32, 2, 128, None), (2, 63, 2, 64, 2, 32, None), (1, 64, 3, 64, 1, 128, None),
    (1, 65, 2, 128, 1, 64, None), (2, 200, 4, 80, 2, 96, (200, 77)), (3, 130, 2, 16, 1, 16, (0, 130, 64)),
    (1, 97, 2, 5, 1, 7, None), (2, 33, 4, 70, 4, 40, (32, 33)), (1, 300, 1, 64, 1, 128, None),
    (3, 150, 1, 24, 1, 128, (-5, 1, 999)), (2, 0, 2, 16, 1, 16, None), (0, 5, 2, 16, 1, 16, None), (1, 3, 2, 1, 2, 1, None),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,H,P,G,N,lengths", CASES)
def test_forward_and_gradients(dev, B, T, H, P, G, N, lengths, dtype):
    x = inputs(dev, B, T, H, P, G, N, dtype, seed=T + N)
    n = None if lengths is None else torch.tensor(lengths, device=dev)
    clean = dict(x)
    if n is not None:  # rows behind a length are not read
        dead = torch.arange(T, device=dev) >= n.clamp(0, T)[:, None]
        for k in ("keys", "values", "queries"):
            x[k] = x[k].masked_fill(dead[..., None, None], float("nan"))
        for k in ("strengths", "log_decays"):
            x[k] = x[k].masked_fill(dead[..., None], float("inf"))
    hidden, memory = run(x, n)
    assert hidden.dtype == dtype and memory.dtype == torch.float32
    ref = oracle.to64(*(clean[k] for k in NAMES), grad=True)
    rh, rm = (t.clone() for t in oracle.delta_scan(*ref, n)) if B else (ref[1] * 1, ref[5] * 1)
    near(hidden, rh, dtype, tol(T, dtype), "hidden")
    near(memory, rm, torch.float32, tol(T, torch.float32), "memory")
    leaves = [x[k].detach().requires_grad_() for k in NAMES]
    out = cuda_ops.cuda_delta_scan(*leaves, lengths=n)
    assert torch.equal(out[0], hidden) and torch.equal(out[1], memory)
    g = torch.Generator().manual_seed(5)
    gh, gm = torch.randn(hidden.shape, generator=g).to(dtype).to(dev), torch.randn(memory.shape, generator=g).to(dev)
    got = torch.autograd.grad(out, leaves, (gh, gm))
    if not B:
        return
    want = torch.autograd.grad((rh, rm), ref, (gh.double().cpu(), gm.double().cpu()), allow_unused=True)
    for k, a, b in zip(NAMES, got, want):
        per_token = k in ("strengths", "log_decays")
        b = torch.zeros(a.shape, dtype=torch.float64) if b is None else b
        rel = 4 * tol(T, a.dtype) * (math.sqrt(P * N) if per_token else 1)
        near(a, b, a.dtype, rel, "gradient of " + k)
        if n is not None and k != "memory":
            assert not a.masked_fill(~dead.reshape(B, T, *[1] * (a.ndim - 2)), 0).any(), k


@pytest.mark.parametrize("dtype", DTYPES)
def test_time_parts(dev, dtype):
    """A few heads over a long sequence, cut in time; lengths end inside, before and behind parts."""
    x = inputs(dev, 3, 2100, 1, 16, 1, 24, dtype, seed=3)
    x["log_decays"] = x["log_decays"] * 0.05
    for n in (None, torch.tensor([2100, 700, 3], device=dev), torch.tensor([0, 1, 64], device=dev)):
        hidden, memory = run(x, n)
        rh, rm = oracle.delta_scan(*oracle.to64(*(x[k] for k in NAMES)), n)
        near(hidden, rh, dtype, tol(2100, dtype), "hidden")
        near(memory, rm, torch.float32, tol(2100, torch.float32), "memory")


def test_types_of_strengths_and_decays(dev):
    for s, d in ((torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32)):
        x = inputs(dev, 1, 70, 2, 32, 1, 32, torch.bfloat16, 1, sdtype=s, ddtype=d)
        leaves = [x[k].detach().requires_grad_() for k in NAMES]
        out = cuda_ops.cuda_delta_scan(*leaves)
        got = torch.autograd.grad(out[0].float().sum() + out[1].sum(), leaves)
        assert [a.dtype for a in got] == [a.dtype for a in leaves]
        rh, _ = oracle.delta_scan(*oracle.to64(*(x[k] for k in NAMES)), None)
        near(out[0], rh, torch.bfloat16, tol(70, torch.bfloat16), "hidden")


def test_without_the_optional_inputs(dev):
    x = inputs(dev, 2, 70, 2, 16, 1, 32, torch.float32, seed=1)
    for gone in (("memory",), ("log_decays",), ("memory", "log_decays")):
        y = dict(x, **{k: None for k in gone})
        leaves = [None if y[k] is None else y[k].detach().requires_grad_() for k in NAMES]
        out = cuda_ops.cuda_delta_scan(*leaves)
        ref = oracle.to64(*(y[k] for k in NAMES), grad=True)
        want = oracle.delta_scan(*ref, None)
        near(out[0], want[0], torch.float32, tol(70, torch.float32), "hidden")
        near(out[1], want[1], torch.float32, tol(70, torch.float32), "memory")
        some = [k for k in NAMES if y[k] is not None]
        # only one of the two outputs has a gradient
        for i in (0, 1):
            fresh = cuda_ops.cuda_delta_scan(*leaves)[i]
            w = torch.randn_like(fresh)
            got = torch.autograd.grad(fresh, [t for t in leaves if t is not None], w, allow_unused=True)
            exp = torch.autograd.grad(want[i], [t for t in ref if t is not None], w.double().cpu(), allow_unused=True, retain_graph=True)
            for k, a, b in zip(some, got, exp):
                b = torch.zeros(a.shape, dtype=torch.float64) if b is None else b
                near(a, b, torch.float32, 4 * tol(70, torch.float32) * (math.sqrt(16 * 32) if k in ("strengths", "log_decays") else 1), k)


def test_gradients_against_differences(dev):
    """The gradient along a direction against the difference of the definition's losses."""
    x = inputs(dev, 2, 100, 2, 24, 1, 40, torch.float32, seed=9)
    leaves = [x[k].detach().requires_grad_() for k in NAMES]
    out = cuda_ops.cuda_delta_scan(*leaves)
    g = torch.Generator().manual_seed(2)
    wh, wm = (torch.randn(o.shape, generator=g, dtype=torch.float64) for o in out)
    got = torch.autograd.grad(out, leaves, (wh.float().to(dev), wm.float().to(dev)))
    base = oracle.to64(*(x[k] for k in NAMES))

    def loss(args):
        h, m = oracle.delta_scan(*args, None)
        return (h * wh.float().double()).sum() + (m * wm.float().double()).sum()

    for i, k in enumerate(NAMES):
        d = torch.randn(base[i].shape, generator=g, dtype=torch.float64)
        step = 1e-5
        args = list(base)
        args[i] = base[i] + step * d
        up = loss(args)
        args[i] = base[i] - step * d
        diff = (up - loss(args)) / (2 * step)
        mine = (got[i].double().cpu() * d).sum()
        # the difference's own error is of step^2; float32 gradients add their roundings like a random walk
        assert abs(mine - diff) <= 1e-4 * (got[i].double().norm().cpu() * d.norm() / math.sqrt(d.numel()) + abs(diff)), k


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,H,P,G,N", [(1, 8, 64, 8, 64), (5, 6, 33, 2, 7), (3, 2, 128, 1, 128), (2, 2, 200, 1, 30), (4, 1, 1, 1, 1)])
def test_single_tokens(dev, B, H, P, G, N, dtype):
    x = inputs(dev, B, 3, H, P, G, N, dtype, seed=P)
    hidden, memory = run(x)
    state = x["memory"].clone()
    for t in range(3):
        args = [x[k][:, t] for k in NAMES[:5]]
        fresh, moved = cuda_ops.cuda_delta_step(*args, state)
        keep = state.clone()
        out, same = cuda_ops.cuda_delta_step(*args, state, memory_out=state)
        assert same is state and torch.equal(out, fresh) and torch.equal(state, moved)
        ref = oracle.to64(*(a[:, None] for a in args), keep)
        rh, rm = oracle.delta_scan(*ref, None)
        near(out, rh[:, 0], dtype, tol(1, dtype), "hidden")
        near(state, rm, torch.float32, tol(1, torch.float32), "memory")
        other = torch.empty_like(keep)
        assert cuda_ops.cuda_delta_step(*args, keep, memory_out=other)[1] is other and torch.equal(other, moved)
    near(state, memory.double().cpu(), torch.float32, 2 * tol(3, torch.float32), "steps and scan")
    no_decay = cuda_ops.cuda_delta_step(*[x[k][:, 0] for k in NAMES[:4]], None, x["memory"])
    zero = cuda_ops.cuda_delta_step(*[x[k][:, 0] for k in NAMES[:4]], torch.zeros(B, H, device=dev), x["memory"])
    assert all(torch.equal(a, b) for a, b in zip(no_decay, zero))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("N", [32, 128])
def test_values_that_are_no_numbers(dev, N, dtype):
    """From its token on, what depends on an infinity or a NaN is NaN; all else is what it was."""
    T, at = 150, 77
    x = inputs(dev, 1, T, 2, 40, 1, N, dtype, seed=4)
    hidden, memory = run(x)
    for bad in (float("inf"), float("-inf"), float("nan")):
        for name, where in (("values", (0, at, 1, 5)), ("queries", (0, at, 0, 3)), ("keys", (0, at, 0, 3)), ("strengths", (0, at, 1)),
                            ("log_decays", (0, at, 1)), ("memory", (0, 1, 5, 3))):
            if name == "log_decays" and bad == float("-inf"):
                continue
            y = dict(x, **{name: x[name].clone()})
            y[name][where] = bad
            h, m = run(y)
            mask = torch.zeros_like(h, dtype=torch.bool)
            gone = torch.zeros_like(m, dtype=torch.bool)
            if name == "values":
                mask[:, at:, 1, 5], gone[:, 1, 5] = True, True
            elif name == "queries":
                mask[:, at] = True
            elif name == "memory":
                mask[:, :, 1, 5], gone[:, 1, 5] = True, True
            elif name == "keys":
                mask[:, at:], gone[:] = True, True
            else:
                mask[:, at:, 1], gone[:, 1] = True, True
            assert torch.equal(torch.isnan(h), mask), (name, bad)
            assert torch.equal(torch.isnan(m), gone), (name, bad)
            assert torch.equal(h[~mask], hidden[~mask]) and torch.equal(m[~gone], memory[~gone]), (name, bad)


def test_a_decay_of_zero_forgets(dev):
    x = inputs(dev, 1, 100, 1, 16, 1, 32, torch.float32, seed=2)
    x["log_decays"][0, 40, 0] = float("-inf")
    x["log_decays"][0, 80, 0] = -3e38
    hidden, memory = run(x)
    rh, rm = oracle.delta_scan(*oracle.to64(*(x[k] for k in NAMES)), None)
    near(hidden, rh, torch.float32, tol(100, torch.float32), "hidden")
    near(memory, rm, torch.float32, tol(100, torch.float32), "memory")
    leaves = [x[k].detach().requires_grad_() for k in NAMES]
    got = torch.autograd.grad(cuda_ops.cuda_delta_scan(*leaves), leaves, (torch.ones_like(hidden), torch.ones_like(memory)))
    assert all(torch.isfinite(t).all() for t in got)


def test_same_keys_again_and_again(dev):
    """Nearly equal keys at full strength, where the chunk's system is worst to invert by powers."""
    x = inputs(dev, 1, 128, 1, 32, 1, 64, torch.float32, seed=6)
    x["keys"] = torch.nn.functional.normalize(x["keys"][:, :1] + 1e-3 * x["keys"], dim=-1) * 0.999
    x["strengths"] = torch.ones_like(x["strengths"])
    x["log_decays"] = torch.zeros_like(x["log_decays"])
    hidden, memory = run(x)
    rh, rm = oracle.delta_scan(*oracle.to64(*(x[k] for k in NAMES)), None)
    near(hidden, rh, torch.float32, 8 * tol(128, torch.float32), "hidden")  # (the misses cancel by the keys' likeness: 8 = sqrt(64))
    near(memory, rm, torch.float32, 8 * tol(128, torch.float32), "memory")


def test_orders_and_slices(dev):
    """Other orders and broadcast rows give what contiguous ones give."""
    x = inputs(dev, 2, 90, 4, 24, 2, 40, torch.bfloat16, seed=7)
    want = run(x)
    y = dict(x)
    y["keys"] = x["keys"].transpose(1, 2).contiguous().transpose(1, 2)
    y["values"] = x["values"].permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0)
    y["strengths"] = x["strengths"].transpose(0, 1).contiguous().transpose(0, 1)
    y["memory"] = x["memory"].transpose(2, 3).contiguous().transpose(2, 3)
    assert all(torch.equal(a, b) for a, b in zip(run(y), want))
    one = x["queries"][:, :1].expand_as(x["queries"])
    leaf = x["queries"][:, :1].clone().requires_grad_()
    got = cuda_ops.cuda_delta_scan(x["keys"], x["values"], leaf.expand_as(x["queries"]), x["strengths"], x["log_decays"], x["memory"])
    assert torch.equal(got[0], run(dict(x, queries=one))[0])
    (grad,) = torch.autograd.grad(got[0].float().sum(), leaf)
    assert grad.shape == leaf.shape and torch.isfinite(grad.float()).all()


def test_rows_past_31_bits(dev):
    """Sequences whose rows begin more than 2^31 elements into their tensor."""
    wide = torch.zeros(2, (1 << 30) + 4096, dtype=torch.bfloat16, device=dev)
    x = inputs(dev, 2, 70, 2, 32, 1, 32, torch.bfloat16, seed=8)
    v = wide[:, -70 * 64:].view(2, 70, 2, 32)
    v.copy_(x["values"])
    assert v.stride(0) > 1 << 30
    far = torch.as_strided(wide.view(-1), (2, 70, 2, 32), ((1 << 30) + 4096, 64, 32, 1), wide.size(1) - 70 * 64)
    assert all(torch.equal(a, b) for a, b in zip(run(dict(x, values=far)), run(x)))


def test_streams_and_repeats(dev):
    """The same bits on every run, on another stream and beside other work."""
    x = inputs(dev, 2, 500, 4, 64, 2, 64, torch.bfloat16, seed=11)
    leaves = [x[k].detach().requires_grad_() for k in NAMES]

    def both():
        out = cuda_ops.cuda_delta_scan(*leaves)
        return (*out, *torch.autograd.grad(out, leaves, (torch.ones_like(out[0]), torch.ones_like(out[1]))))

    want = both()
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for s in side:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(both())
    for s in side:
        torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    for other in got + [both()]:
        assert all(torch.equal(a, b) for a, b in zip(other, want))


def test_captured_and_replayed(dev):
    """A graph of a prompt, its norm and steps in place, replayed with eager work in between."""
    x = inputs(dev, 2, 130, 2, 32, 1, 32, torch.bfloat16, seed=12)
    state = x["memory"].clone()
    token = [x[k][:, 0].clone() for k in NAMES[:5]]

    def work():
        h, m = run(x)
        n = cuda_ops.cuda_group_norm(h.flatten(-2), 2, activation="silu", center=False)
        out, _ = cuda_ops.cuda_delta_step(*token, state, memory_out=state)
        return h, m, n, out

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work()
    for i in range(4):
        state.copy_(x["memory"])
        x["keys"].copy_(torch.nn.functional.normalize(torch.randn_like(x["keys"].float()), dim=-1))
        graph.replay()
        torch.cuda.synchronize()
        after = state.clone()
        state.copy_(x["memory"])
        assert all(torch.equal(a, b) for a, b in zip(got, work()))
        assert torch.equal(state, after)


def test_version_of_a_given_state(dev):
    x = inputs(dev, 1, 1, 1, 8, 1, 8, torch.float32, seed=1)
    state = x["memory"].clone()
    w = torch.ones_like(state, requires_grad=True)
    loss = (w * state).sum()
    cuda_ops.cuda_delta_step(*[x[k][:, 0] for k in NAMES[:5]], state, memory_out=state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        made = torch.zeros(1, 1, 8, 8, device=dev)
    cuda_ops.cuda_delta_step(*[x[k][:, 0] for k in NAMES[:5]], made, memory_out=made)


def test_refusals(dev):
    x = inputs(dev, 2, 5, 4, 16, 2, 16, torch.bfloat16, seed=1)
    call = lambda **k: run(dict(x, **k))  # noqa: E731
    for kw, match in [
            (dict(keys=x["keys"][:, :4]), "agree"), (dict(queries=x["queries"][..., :8]), "agree"),
            (dict(values=x["values"].float()), "share a type"), (dict(strengths=x["strengths"][..., :3]), "agree"),
            (dict(strengths=x["strengths"].half()), "share a type"), (dict(log_decays=x["log_decays"].double()), "float32"),
            (dict(memory=x["memory"][:, :, :8]), "memory must be"), (dict(keys=x["keys"][:, :, 0]), "must be"),
            (dict(memory=x["memory"].cpu()), "must be on"), (dict(log_decays=x["log_decays"][:1]), "agree")]:
        with pytest.raises(ValueError, match=match):
            call(**kw)
    big = torch.zeros(1, 2, 1, 129, device=dev)
    with pytest.raises(ValueError, match="key_dim"):
        cuda_ops.cuda_delta_scan(big, torch.zeros(1, 2, 1, 4, device=dev), big, torch.zeros(1, 2, 1, device=dev))
    with pytest.raises(ValueError, match="lengths"):
        run(x, torch.zeros(3, dtype=torch.long, device=dev))
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        run({k: v.double() for k, v in x.items()})
    with pytest.raises(RuntimeError, match="forward"):
        import torch.autograd.forward_ad as fwd
        with fwd.dual_level():
            run(dict(x, memory=fwd.make_dual(x["memory"], torch.ones_like(x["memory"]))))
    leaf = x["values"].detach().requires_grad_()
    out = run(dict(x, values=leaf))[0]
    (g,) = torch.autograd.grad(out.float().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().sum().backward()
    step = [x[k][:, 0] for k in NAMES[:5]]
    with pytest.raises(ValueError, match="gradients"):
        cuda_ops.cuda_delta_step(*step, x["memory"].requires_grad_(), memory_out=torch.empty_like(x["memory"]))
    with pytest.raises(ValueError, match="contiguous"):
        cuda_ops.cuda_delta_step(*step, x["memory"].detach(), memory_out=torch.empty(2, 4, 16, 17, device=dev)[..., 1:])
    pool = torch.zeros(2 * 4 * 16 * 16 + 64, device=dev)
    a, b = pool[:2048].view(2, 4, 16, 16), pool[64:64 + 2048].view(2, 4, 16, 16)
    with pytest.raises(RuntimeError, match="overlap"):
        cuda_ops.cuda_delta_step(*step, a, memory_out=b)
