"""Forward-mode derivatives of the entry points that choose their path by whether a gradient is wanted: carried by the
PyTorch form or refused by the autograd function, never dropped by the native op alone."""

import pytest
import torch

from rnn_with_grm_amd import cuda_ops as ops

pytestmark = pytest.mark.gpu


def cases(dev):
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g).to(dev)  # noqa: E731
    mem, idx = r(2, 3, 8, 4), torch.randint(0, 3, (2, 5, 2), generator=g).to(dev)
    w, ln = r(12, 16), r(12)
    return {
        "gather_apply": (lambda t: ops.cuda_gather_apply(mem, idx, t), r(2, 5, 4)),
        "retrieve_fuse": (lambda t: ops.cuda_retrieve_fuse(mem, idx, t, torch.ones(2, 5, 2, device=dev), torch.ones(2, 5, 8, device=dev)), r(2, 5, 4)),
        "project_split": (lambda t: ops.cuda_project_split(t, 4, 4)[0], r(2, 5, 12)),
        "project_gemm": (lambda t: ops.cuda_project_gemm(t, w, None, 4, 4)[0], r(2, 5, 16)),
        "residual_layer_norm": (lambda t: ops.cuda_residual_layer_norm(t, t * 0.5, ln, ln), r(2, 5, 12)),
        "linear_residual_layer_norm": (lambda t: ops.cuda_linear_residual_layer_norm(t, w, ln, torch.ones(2, 5, 12, device=dev), ln, ln), r(2, 5, 16)),
    }


@pytest.mark.parametrize("name", ["gather_apply", "retrieve_fuse", "project_split", "project_gemm", "residual_layer_norm",
                                  "linear_residual_layer_norm"])
def test_tangents(dev, name):
    f, t = cases(dev)[name]
    tangent = torch.randn_like(t)
    with torch.no_grad():
        want = (f(t + 0.01 * tangent) - f(t - 0.01 * tangent)) / 0.02
    try:
        _, moved = torch.func.jvp(f, (t,), (tangent,))
    except (RuntimeError, NotImplementedError):
        return
    # Central differences over 0.01 of a tangent of order 1: 1e-4 of third derivatives of order 1 to 10, and float32's
    # (with float16 rows inside, 2^-11) rounding over 0.02.
    assert (moved - want).norm() <= 0.1 * want.norm()
