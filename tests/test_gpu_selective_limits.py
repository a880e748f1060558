"""The largest sizes that the selective scan and its single token take."""

import pytest
import torch

from rnn_with_grm_amd import cuda_ops

pytestmark = pytest.mark.gpu


def one_token(dev, B, H, P, N, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    return dict(keys=r(B, 1, N), values=r(B, H, P), queries=r(B, 1, N), steps=r(B, H).abs() * 0.1, rates=-torch.ones(H, device=dev),
                memory=r(B, H, P, N))


def check(x, hidden, memory):
    """One token in float32: two products and a sum of N, against the same in float64."""
    d = x["steps"].double()
    k, q = x["keys"].double()[:, :, None], x["queries"].double()[:, :, None]
    want = torch.exp(-d)[..., None, None] * x["memory"].double() + (d[..., None] * x["values"].double())[..., None] * k
    torch.testing.assert_close(memory.double(), want, rtol=1e-5, atol=1e-5)
    mag = (want.abs() * q.abs()).sum(-1)
    assert ((hidden.double() - (want * q).sum(-1)).abs() <= (want.shape[-1] + 8) * 2.0 ** -24 * (mag + 1)).all()


def test_as_many_sequences_as_a_grid_takes(dev):
    x = one_token(dev, (1 << 23) - 1, 1, 1, 1, 1)
    args = [x[k][:, None] for k in ("keys", "values", "queries", "steps")]
    hidden, memory = cuda_ops.cuda_selective_scan(*args, x["rates"], x["memory"])
    check(x, hidden[:, 0], memory)
    check(x, *cuda_ops.cuda_selective_step(*(x[k] for k in ("keys", "values", "queries", "steps", "rates", "memory"))))
    wide = {k: v if k == "rates" else torch.cat([v, v[:1]]) for k, v in x.items()}
    with pytest.raises(RuntimeError, match="below 8388608"):
        cuda_ops.cuda_selective_scan(*(wide[k][:, None] for k in ("keys", "values", "queries", "steps")), x["rates"], wide["memory"])


def test_a_token_of_the_most_value_rows(dev):
    """More tiles of rows than a grid's second dimension has."""
    x = one_token(dev, 1, 1, 1 << 21, 65, 2)
    hidden, memory = cuda_ops.cuda_selective_step(*(x[k] for k in ("keys", "values", "queries", "steps", "rates", "memory")))
    check(x, hidden, memory)
