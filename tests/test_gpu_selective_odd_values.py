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
