"""Selective state scan on the GPU against its float64 definition.

Tolerances.  ``mag`` is the definition on absolute values: the sum of the magnitudes of everything that
is added up.  Float32 arithmetic: a result is a sum of up to N + 64 products a chunk of at most 64
tokens, and the state passes T / 32 chunks or fewer of four roundings each, so it is off by at most
(N + 2 * 64 + T / 8 + 32) 2^-24 of mag, the exponentials' few steps included (float32 and float16 inputs run so).
bfloat16 inputs: the state a query reads, or the weight between two tokens, is rounded once more to
bfloat16, half a step of each term, so half a step of mag.  Last, the output's own rounding: half a
step of its value."""

import pytest
import torch

import selective_oracle as oracle
from rnn_with_grm_amd import cuda_ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def half(dtype):
    return torch.finfo(dtype).eps / 2


def inputs(dev, B, T, H, P, G, N, dtype, seed, steps_dtype=None, wide=True):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    rows = r(B, T, H * P + 2 * G * N + (8 if wide else 0)).to(dtype).to(dev)
    return dict(keys=rows[..., H * P:H * P + G * N].unflatten(-1, (G, N)),
                values=rows[..., :H * P].unflatten(-1, (H, P)),
                queries=rows[..., H * P + G * N:H * P + 2 * G * N].unflatten(-1, (G, N)),
                steps=(r(B, T, H) - 2).to(steps_dtype or dtype).to(dev), rates=-torch.exp(r(H)).to(dev),
                memory=r(B, H, P, N).to(dev), skip=r(H).to(dev), step_bias=(r(H) - 1).to(dev))


NAMES = ("keys", "values", "queries", "steps", "rates", "memory", "skip", "step_bias")


def run(x, lengths=None, softplus=True, fn=None):
    return (fn or cuda_ops.cuda_selective_scan)(
        x["keys"], x["values"], x["queries"], x["steps"], x["rates"], x["memory"], skip=x["skip"],
        step_bias=x["step_bias"], softplus=softplus, lengths=lengths)


def definition(x, lengths, softplus, absolute=False):
    """The float64 result; `absolute`: of the magnitudes, with the decays and step sizes as they are."""
    v = {k: x[k] for k in NAMES}
    if absolute:
        v = {k: t if t is None or k in ("steps", "rates", "step_bias") else t.abs() for k, t in v.items()}
    return oracle.selective_scan(*(v[k] for k in NAMES), lengths, softplus)


def near(got, ref, mag, dtype, rounded, steps):
    got, ref, mag = got.double().cpu(), ref.detach(), mag.detach()
    assert got.shape == ref.shape
    bound = half(dtype) * ref.abs() * 1.001 + (rounded + steps * U) * mag + torch.finfo(dtype).smallest_normal * half(dtype) * 2
    bad = ~((got - ref).abs() <= bound)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {((got - ref).abs() / bound).nan_to_num(99).max():.2f} of the bound"


def check(x, lengths, softplus, dtype):
    hidden, memory = run(x, lengths, softplus)
    assert hidden.dtype == dtype and memory.dtype == torch.float32
    xr = dict(zip(NAMES, oracle.to64(*(x[k] for k in NAMES))))
    ref, rmem = definition(xr, lengths, softplus)
    xr = {k: None if t is None else t.nan_to_num() for k, t in xr.items()}
    mag, mmag = definition(xr, lengths, softplus, absolute=True)
    B, T, H, P = x["values"].shape
    steps = x["keys"].size(-1) + 128 + T / 8 + 32
    near(hidden, ref, mag, dtype, half(dtype) * 1.01 if dtype == torch.bfloat16 else 0, steps)
    near(memory, rmem, mmag, torch.float32, 0, steps)
    return hidden, memory


CASES = [
    # B, T, H, P, G, N, lengths
    (2, 1, 2, 64, 1, 64, None), (1, 2, 4, 32, 2, 128, None), (2, 63, 2, 64, 2, 32, None), (1, 64, 3, 64, 1, 128, None),
    (1, 65, 2, 128, 1, 64, None), (2, 200, 4, 80, 2, 96, (200, 77)), (3, 130, 2, 16, 1, 16, (0, 130, 64)),
    (1, 97, 2, 5, 1, 7, None), (2, 33, 4, 70, 4, 40, (32, 33)), (1, 600, 1, 64, 1, 128, None),
    (3, 150, 1, 24, 1, 128, (-5, 1, 999)), (2, 0, 2, 16, 1, 16, None),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,H,P,G,N,lengths", CASES)
def test_forward(dev, B, T, H, P, G, N, lengths, dtype):
    x = inputs(dev, B, T, H, P, G, N, dtype, seed=T + N)
    n = None if lengths is None else torch.tensor(lengths, device=dev)
    if n is not None:  # rows behind a length are not read
        dead = torch.arange(T, device=dev) >= n.clamp(0, T)[:, None]
        for k in ("keys", "values", "queries"):
            x[k] = x[k].masked_fill(dead[..., None, None], float("nan"))
        x["steps"] = x["steps"].masked_fill(dead[..., None], float("inf"))
    check(x, n, True, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_long_walk_in_parts(dev, dtype):
    """A few heads over a long sequence, cut in time; lengths end inside, before and behind parts."""
    x = inputs(dev, 3, 2100, 1, 16, 1, 24, dtype, seed=3)
    x["rates"] = x["rates"] * 0.02
    check(x, torch.tensor([2100, 700, 3], device=dev), True, dtype)
    check(x, None, True, dtype)


def test_without_the_optional_inputs(dev):
    x = inputs(dev, 2, 70, 2, 16, 1, 32, torch.bfloat16, seed=1, steps_dtype=torch.float32)
    x["step_bias"] = x["step_bias"].abs()  # without softplus a negative step grows the state past float32
    for gone in (("memory",), ("skip",), ("step_bias",), ("memory", "skip", "step_bias")):
        y = dict(x, **{k: None for k in gone})
        y["steps"] = y["steps"].abs() * 0.1
        check(y, None, False, torch.bfloat16)
        check(y, None, True, torch.bfloat16)


def test_strong_decay_and_growth(dev):
    """Decays that underflow within a token, and a state that grows."""
    x = inputs(dev, 1, 100, 2, 16, 1, 16, torch.float32, seed=8)
    x["rates"] = torch.tensor([-1e5, 0.05], device=dev)
    check(x, None, True, torch.float32)


def test_a_reset_leaves_the_next_tokens_their_decay(dev):
    """A token that wipes the state (log decay -1e30) must not hide the decays behind it."""
    x = inputs(dev, 1, 90, 1, 16, 1, 16, torch.float32, seed=9)
    x["steps"], x["step_bias"] = x["steps"].abs() * 0.1, None
    x["steps"][0, 40] = 1e30
    x["values"] = x["values"].clone()
    x["values"][0, 40] = 0
    check(x, None, False, torch.float32)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,H,P,G,N", [(1, 8, 64, 1, 64), (3, 4, 80, 2, 128), (2, 2, 5, 1, 7), (33, 3, 16, 3, 16),
                                       (2, 2, 33, 1, 32), (1, 1, 200, 1, 100)])
def test_step(dev, B, H, P, G, N, dtype):
    x = inputs(dev, B, 1, H, P, G, N, dtype, seed=P)
    xr = dict(zip(NAMES, oracle.to64(*(x[k] for k in NAMES))))
    ref, rmem = definition(xr, None, True)
    mag, mmag = definition(xr, None, True, absolute=True)
    args = [x[k][:, 0] for k in ("keys", "values", "queries", "steps")] + [x["rates"]]
    more = dict(skip=x["skip"], step_bias=x["step_bias"], softplus=True)
    hidden, moved = cuda_ops.cuda_selective_step(*args, x["memory"], **more)
    near(hidden, ref[:, 0], mag[:, 0], dtype, 0, N + 32)
    near(moved, rmem, mmag, torch.float32, 0, 32)
    kept = x["memory"].clone()
    again, same = cuda_ops.cuda_selective_step(*args, kept, memory_out=kept, **more)
    assert same is kept and torch.equal(kept, moved) and torch.equal(again, hidden)


def test_refusals(dev):
    x = inputs(dev, 2, 5, 4, 16, 2, 16, torch.float32, seed=1)
    scan = lambda **kw: run({**x, **kw}, kw.get("lengths"))  # noqa: E731
    for call in (lambda: scan(keys=x["keys"][..., :8]), lambda: scan(keys=x["keys"][:, :3]),
                 lambda: scan(values=x["values"].half()), lambda: scan(values=x["values"][:, :, :3]),
                 lambda: scan(steps=x["steps"][..., :2]), lambda: scan(steps=x["steps"].half()),
                 lambda: scan(rates=x["rates"][:2]), lambda: scan(rates=x["rates"].cpu()),
                 lambda: scan(memory=x["memory"][:1]), lambda: scan(skip=x["skip"][:1]),
                 lambda: scan(step_bias=x["step_bias"][:1]), lambda: scan(keys=x["keys"][:, :, 0]),
                 lambda: scan(lengths=torch.zeros(3, dtype=torch.long, device=dev)),
                 lambda: scan(lengths=torch.zeros(2, device=dev)),
                 lambda: run({k: v.double() for k, v in x.items()}),
                 lambda: scan(keys=torch.zeros(2, 5, 2, 136, device=dev), queries=torch.zeros(2, 5, 2, 136, device=dev),
                              memory=None)):
        with pytest.raises(ValueError):
            call()
    args = [x[k][:, 0] for k in ("keys", "values", "queries", "steps")] + [x["rates"], x["memory"]]
    step = cuda_ops.cuda_selective_step
    for call in (lambda: step(*args, memory_out=x["memory"].half()), lambda: step(*args, memory_out=x["memory"][:1]),
                 lambda: step(*args[:-1], x["memory"].half()), lambda: step(x["keys"], *args[1:]),
                 lambda: step(*args[:-2], x["rates"].clone().requires_grad_(), x["memory"], memory_out=x["memory"])):
        with pytest.raises(ValueError):
            call()
    both = torch.zeros(3, 4, 16, 16, device=dev)
    with pytest.raises(RuntimeError):  # the new state half over the old one
        step(*args[:-1], both[:2], memory_out=both[1:])


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities_and_nan_reach_no_earlier_token(dev, dtype):
    """A value that is no number changes its own row of the state from its token on, and nothing else."""
    x = inputs(dev, 1, 150, 2, 32, 1, 32, dtype, seed=21)
    clean, clean_memory = run(x)
    x["values"] = x["values"].clone()
    x["values"][0, 20, 1, 5] = float("inf")
    x["values"][0, 77, 0, 9] = float("nan")
    hidden, memory = run(x)
    same = torch.ones_like(hidden, dtype=torch.bool)
    same[0, 20:, 1, 5] = False
    same[0, 77:, 0, 9] = False
    assert torch.equal(hidden[same], clean[same])
    assert not torch.isfinite(hidden[0, 20, 1, 5]) and torch.isnan(hidden[0, 77:, 0, 9]).all()
    rows = torch.ones_like(memory, dtype=torch.bool)
    rows[0, 1, 5] = rows[0, 0, 9] = False
    assert torch.equal(memory[rows], clean_memory[rows])


@pytest.mark.parametrize("which", ["keys", "queries", "steps"])
def test_an_odd_key_query_or_step_reaches_no_earlier_token(dev, which):
    x = inputs(dev, 1, 150, 2, 32, 2, 32, torch.bfloat16, seed=22)
    clean, _ = run(x)
    x[which] = x[which].clone()
    if which == "steps":
        x[which][0, 70, 1] = float("nan")
    else:
        x[which][0, 70, 1, 3] = float("nan")
    hidden, _ = run(x)
    assert torch.equal(hidden[0, :70], clean[0, :70]) and torch.equal(hidden[0, :, 0], clean[0, :, 0])
    assert torch.isnan(hidden[0, 70, 1]).all()
    if which == "queries":
        assert torch.equal(hidden[0, 71:], clean[0, 71:])
