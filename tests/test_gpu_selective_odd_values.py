"""Infinities in the selective scan's inputs where the definition's results are numbers or infinities, not NaN."""

import pytest
import torch

import selective_oracle as oracle
from rnn_with_grm_amd import cuda_ops
from test_gpu_selective_scan import DTYPES, NAMES, definition, inputs, run

pytestmark = pytest.mark.gpu


def same_kinds(got, want):
    for kind in (torch.isposinf, torch.isneginf, torch.isnan):
        assert torch.equal(kind(got).cpu(), kind(want)), kind.__name__


@pytest.mark.parametrize("dtype", DTYPES)
def test_an_infinite_value_without_skip(dev, dtype):
    x = inputs(dev, 1, 40, 2, 16, 1, 16, dtype, seed=5)
    x["keys"], x["queries"], x["values"], x["skip"] = x["keys"].abs() + 0.125, x["queries"].abs() + 0.125, x["values"].clone(), None
    x["rates"] = x["rates"].clamp(min=-0.05)
    x["values"][0, 0, 1, 3], x["values"][0, 7, 0, 2] = float("inf"), float("-inf")
    ref, rmem = definition(dict(zip(NAMES, oracle.to64(*(x[k] for k in NAMES)))), None, True)
    assert int(torch.isinf(ref).sum()) == 40 + 33 and not torch.isnan(ref).any()
    hidden, memory = run(x)
    same_kinds(hidden, ref), same_kinds(memory, rmem)
    y, moved = cuda_ops.cuda_selective_step(*(x[k][:, 0] for k in ("keys", "values", "queries", "steps")), x["rates"], x["memory"],
                                            step_bias=x["step_bias"], softplus=True)
    same_kinds(y, ref[:, 0])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,lengths", [(70, None), (200, (200, 77))])
def test_a_rate_of_minus_infinity(dev, dtype, T, lengths):
    """A head that forgets everything at every token: M_t = d_t v_t k_t^T, whatever its number of tokens; the tokens behind a
    length leave the state alone.  The other head as without it."""
    x = inputs(dev, 2, T, 2, 16, 1, 16, dtype, seed=6)
    n = None if lengths is None else torch.tensor(lengths, device=dev)
    clean = run(x, n)
    x["rates"] = torch.stack([x["rates"][0], torch.tensor(float("-inf"), device=dev)])
    hidden, memory = run(x, n)
    assert torch.equal(hidden[:, :, 0], clean[0][:, :, 0]) and torch.equal(memory[:, 0], clean[1][:, 0])
    for b in range(2):
        last = (T if n is None else lengths[b]) - 1
        d = torch.nn.functional.softplus(x["steps"][b, :, 1].double() + x["step_bias"][1].double())[:, None]
        v, k, q = (x[s][b, :, -1].double() for s in ("values", "keys", "queries"))
        want = d * (k * q).sum(-1, keepdim=True) * v + x["skip"][1].double() * v
        mag = d * (k * q).abs().sum(-1, keepdim=True) * v.abs() + (x["skip"][1] * v).abs()
        off = (hidden[b, :last + 1, 1].double() - want[:last + 1]).abs()
        e = torch.finfo(dtype).eps / 2 if dtype != torch.float32 else 0
        assert (off <= e * 1.01 * want[:last + 1].abs() + (2.0 ** -16 * 1.01 * (dtype == torch.bfloat16) + 64 * 2.0 ** -24) * mag[:last + 1] + 1e-7).all()
        torch.testing.assert_close(memory[b, 1].double(), d[last] * v[last][:, None] * k[last], rtol=1e-5, atol=1e-6)
        assert (hidden[b, last + 1:] == 0).all()
