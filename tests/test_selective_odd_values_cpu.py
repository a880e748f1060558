"""Infinities and NaN in the PyTorch forms of the selective scan and the short convolution: what reaches what."""

import pytest
import torch

from rnn_with_grm_amd import cuda_ops

INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("W", [2, 3, 4])
def test_an_infinity_before_a_length_in_the_weights_gradient(W):
    g = torch.Generator().manual_seed(1)
    x, w, st = torch.randn(1, 9, 3, generator=g), torch.randn(3, W, generator=g).requires_grad_(), torch.randn(1, W - 1, 3, generator=g)
    x[0, 5, 1] = INF
    out, _ = cuda_ops.cuda_short_conv(x, w, None, st, lengths=torch.tensor([6]))
    (dw,) = torch.autograd.grad(out.sum(), w)
    odd = torch.zeros(3, W, dtype=torch.bool)
    odd[1, W - 1] = True  # only its own token's gradient meets it
    assert torch.equal(torch.isinf(dw), odd) and not torch.isnan(dw).any()


NAMES = ("keys", "values", "queries", "steps", "rates", "memory", "skip", "step_bias")


def scan_inputs(T=10, H=2, P=3, G=1, N=4):
    g = torch.Generator().manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return dict(keys=r(1, T, G, N), values=r(1, T, H, P), queries=r(1, T, G, N), steps=r(1, T, H) - 2, rates=-torch.exp(r(H)),
                memory=r(1, H, P, N), skip=r(H), step_bias=r(H) - 1)


def scan(x, **kw):
    return cuda_ops.cuda_selective_scan(*(x[k] for k in NAMES[:6]), skip=x["skip"], step_bias=x["step_bias"], softplus=True, **kw)


@pytest.mark.parametrize("T", [10, 70])  # in one chunk, and in the second of two
@pytest.mark.parametrize("which", ["keys", "values", "queries", "steps"])
@pytest.mark.parametrize("odd", [INF, -INF, NAN])
def test_nothing_odd_reaches_an_earlier_token(which, odd, T):
    x = scan_inputs(T)
    clean, _ = scan(x)
    x[which] = x[which].clone()
    x[which][(0, T - 3, 0) + (() if which == "steps" else (1,))] = odd
    hidden, _ = scan(x)
    assert torch.equal(hidden[:, :T - 3], clean[:, :T - 3])
    if which == "values":  # and only its own row of the state
        same = torch.ones_like(hidden, dtype=torch.bool)
        same[0, T - 3:, 0, 1] = False
        torch.testing.assert_close(hidden[same], clean[same])
    if which == "queries":
        assert torch.equal(hidden[:, T - 2:], clean[:, T - 2:])


def test_infinite_values_as_the_definition_sums_them():
    """Signs of infinite sums, infinities of both signs, and a token whose weight for one is zero."""
    x = scan_inputs()
    x["keys"], x["queries"] = x["keys"].abs() + 0.1, x["queries"].abs() + 0.1
    x["values"] = x["values"].clone()
    x["values"][0, 2, 0, 0], x["values"][0, 4, 1, 1], x["values"][0, 6, 1, 1] = INF, -INF, INF
    x["skip"] = x["skip"].abs()
    import selective_oracle as oracle
    ref, rmem = oracle.selective_scan(*(x[k].double() for k in NAMES), None, True)
    hidden, memory = scan(x)
    for kind in (torch.isposinf, torch.isneginf, torch.isnan):
        assert torch.equal(kind(hidden), kind(ref)) and torch.equal(kind(memory), kind(rmem))
    fine = torch.isfinite(ref)
    torch.testing.assert_close(hidden[fine].double(), ref[fine], rtol=1e-4, atol=1e-5)


def test_under_vmap():
    """The check for odd values asks nothing that vmap cannot answer."""
    x = scan_inputs()
    several = torch.randn(3, *x["values"].shape, generator=torch.Generator().manual_seed(5))
    out = torch.func.vmap(lambda v: scan({**x, "values": v})[0])(several)
    for o, v in zip(out, several):
        torch.testing.assert_close(o, scan({**x, "values": v})[0])
    jac = torch.func.jacfwd(lambda r: scan({**x, "rates": r})[0])(x["rates"])
    assert jac.shape == (1, 10, 2, 3, 2) and torch.isfinite(jac).all()


@pytest.mark.parametrize("T,lengths", [(10, None), (70, None), (70, (41,))])
def test_a_rate_of_minus_infinity(T, lengths):
    """A head that forgets everything at every token."""
    import selective_oracle as oracle
    x = {k: v.double() for k, v in scan_inputs(T).items()}
    x["rates"] = torch.tensor([-0.5, -INF], dtype=torch.float64)
    n = None if lengths is None else torch.tensor(lengths)
    got = scan(x, lengths=n)
    for a, b in zip(got, oracle.selective_scan(*(x[k] for k in NAMES), n, True)):
        torch.testing.assert_close(a, b, rtol=1e-10, atol=1e-10)
