"""What the selective scan and the short convolution tell autograd."""

import pytest
import torch

from rnn_with_grm_amd import cuda_ops
from test_gpu_selective_scan import NAMES, inputs, run

pytestmark = pytest.mark.gpu


def test_the_first_state_may_be_moved_before_the_backward(dev):
    """The scan's backward does not read the first state, so a caller that keeps one buffer may overwrite it."""
    x = inputs(dev, 2, 70, 2, 16, 1, 16, torch.float32, seed=2)
    leaves = {k: (x[k] if k == "memory" else x[k].detach().requires_grad_()) for k in NAMES}
    names = [k for k in NAMES if k != "memory"]
    want = torch.autograd.grad(run(leaves)[0].sum(), [leaves[k] for k in names])
    hidden, memory = run(leaves)
    leaves["memory"].copy_(memory.detach())
    got = torch.autograd.grad(hidden.sum(), [leaves[k] for k in names])
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def step_args(x):
    return [x[k][:, 0] for k in ("keys", "values", "queries", "steps")] + [x["rates"]]


def test_steps_in_place_count_as_writes(dev):
    """A state that a graph has saved for its backward and a single token has moved since: the backward is refused, as
    after any write in place, and not computed from the moved state."""
    g = torch.Generator().manual_seed(3)
    x, w, state = (torch.randn(*s, generator=g).to(dev) for s in ((2, 9, 8), (8, 4), (2, 3, 8)))
    w.requires_grad_()
    out, _ = cuda_ops.cuda_short_conv(x, w, None, state)
    with torch.no_grad():
        cuda_ops.cuda_short_conv_step(x[:, 0], state, w, state_out=state)
    assert state._version == 1
    with pytest.raises(RuntimeError, match="inplace"):
        out.sum().backward()
    a = inputs(dev, 2, 1, 2, 16, 1, 16, torch.float32, seed=4)
    leaf = torch.ones_like(a["memory"], requires_grad=True)
    product = (leaf * a["memory"]).sum()  # saves the state
    cuda_ops.cuda_selective_step(*step_args(a), a["memory"], memory_out=a["memory"])
    assert a["memory"]._version == 1
    with pytest.raises(RuntimeError, match="inplace"):
        product.backward()


def test_steps_in_place_in_inference_mode(dev):
    with torch.inference_mode():
        a = inputs(dev, 2, 1, 2, 16, 1, 16, torch.float32, seed=4)
        want = cuda_ops.cuda_selective_step(*step_args(a), a["memory"])
        got = cuda_ops.cuda_selective_step(*step_args(a), a["memory"], memory_out=a["memory"])
    assert all(torch.equal(u, v) for u, v in zip(got, want)) and got[1] is a["memory"]


@pytest.mark.parametrize("grad_enabled", [True, False])
def test_no_forward_derivatives(dev, grad_enabled):
    """A tangent is refused, not dropped; the PyTorch forms carry it."""
    x = inputs(dev, 2, 5, 2, 16, 1, 16, torch.float32, seed=5)
    c, w, state = torch.randn(2, 5, 8, device=dev), torch.randn(8, 4, device=dev), torch.randn(2, 3, 8, device=dev)
    calls = {
        "conv": (lambda t, **k: cuda_ops.cuda_short_conv(t, w, None, state, **k)[0], c),
        "conv_step": (lambda t, **k: cuda_ops.cuda_short_conv_step(c[:, 0], t, w, **k)[1], state),
        "scan": (lambda t, **k: cuda_ops.cuda_selective_scan(x["keys"], x["values"], x["queries"], x["steps"], t, **k)[0],
                 x["rates"]),
        "step": (lambda t, **k: cuda_ops.cuda_selective_step(*step_args(x), t, **k)[0], x["memory"]),
    }
    with torch.set_grad_enabled(grad_enabled):
        for name, (f, t) in calls.items():
            tangent = torch.randn_like(t)
            for mode in (lambda g: torch.func.jvp(g, (t,), (tangent,)), lambda g: forward(g, t, tangent)):
                with pytest.raises((RuntimeError, NotImplementedError)):
                    mode(f)
            out, moved = torch.func.jvp(lambda v: f(v, enabled=False), (t,), (tangent,))
            plain = (f(t + 0.01 * tangent, enabled=False) - f(t - 0.01 * tangent, enabled=False)) / 0.02
            assert (moved - plain).norm() <= 0.02 * plain.norm(), name  # differences over 0.01 of a tangent of order 1
            with torch.no_grad():
                assert torch.isfinite(f(t)).all()  # and without one the kernels run


def forward(g, t, tangent):
    with torch.autograd.forward_ad.dual_level():
        return g(torch.autograd.forward_ad.make_dual(t, tangent))


def test_steps_on_states_made_in_inference_mode(dev):
    """A prompt in inference mode, its single tokens outside of it, in place."""
    g = torch.Generator().manual_seed(6)
    x, w = torch.randn(2, 9, 8, generator=g).to(dev), torch.randn(8, 4, generator=g).to(dev)
    a = inputs(dev, 2, 1, 2, 16, 1, 16, torch.float32, seed=6)
    with torch.inference_mode():
        _, state = cuda_ops.cuda_short_conv(x, w)
        _, memory = run(a)
    kept = state.clone(), memory.clone()
    with torch.no_grad():
        want = cuda_ops.cuda_short_conv_step(x[:, 0], kept[0], w), cuda_ops.cuda_selective_step(*step_args(a), kept[1])
        y, _ = cuda_ops.cuda_short_conv_step(x[:, 0], state, w, state_out=state)
        h, _ = cuda_ops.cuda_selective_step(*step_args(a), memory, memory_out=memory)
    assert torch.equal(y, want[0][0]) and torch.equal(state, want[0][1])
    assert torch.equal(h, want[1][0]) and torch.equal(memory, want[1][1])
