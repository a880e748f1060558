"""The delta rule's C entry points with inputs, outputs and gradients that begin anywhere (states and workspaces are 16-byte
aligned, as the header says): the results are those of aligned ones, since only the width of loads and stores changes."""

import ctypes

import pytest
import torch

from rnn_with_grm_amd import capi

pytestmark = pytest.mark.gpu
B, T, H, P, N = 2, 150, 4, 48, 64


def arguments(x, dtype, G):
    a = capi.DeltaArgs()
    for k in ("keys", "values", "queries", "strengths", "log_decays"):
        setattr(a, k, x[k].data_ptr())
    sizes = dict(batch=B, seq_len=T, heads=H, value_dim=P, groups=G, key_dim=N, keys_batch_stride=T * G * N, keys_token_stride=G * N,
                 values_batch_stride=T * H * P, values_token_stride=H * P, queries_batch_stride=T * G * N, queries_token_stride=G * N,
                 strengths_batch_stride=T * H, strengths_token_stride=H, decays_batch_stride=T * H, decays_token_stride=H,
                 dtype=dtype, strengths_dtype=dtype, decays_dtype=dtype)
    for k, v in sizes.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("dtype,code", [(torch.bfloat16, capi.BF16), (torch.float32, capi.F32), (torch.float16, capi.F16)])
@pytest.mark.parametrize("G", [2, 4])  # (heads of a group in shares, and a head a group)
def test_buffers_that_begin_anywhere(dev, G, dtype, code):
    g = torch.Generator().manual_seed(1)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    unit = lambda: torch.nn.functional.normalize(r(B, T, G, N), dim=-1)  # noqa: E731
    base = dict(keys=unit(), values=r(B, T, H, P), queries=unit(), strengths=torch.rand(B, T, H, generator=g),
                log_decays=-0.1 * torch.rand(B, T, H, generator=g), grad_hidden=r(B, T, H, P))
    base = {k: v.to(dtype).to(dev) for k, v in base.items()}
    lib = capi.load()
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)

    def buffer(shape, dt, shift):
        return torch.zeros(shape.numel() + 64, dtype=dt, device=dev)[shift:shift + shape.numel()].view(shape)

    def both(shifted):
        at = lambda name: 1 if name in shifted else 0  # noqa: E731
        x = {}
        for k, v in base.items():
            x[k] = buffer(v.shape, dtype, at(k))
            x[k].copy_(v)
        a = arguments(x, code, G)
        out = {"hidden": buffer(base["values"].shape, dtype, at("hidden")), "miss": buffer(base["values"].shape, torch.float32, at("miss"))}
        for k in ("keys", "values", "queries", "strengths", "log_decays"):
            out["grad_" + k] = buffer(base[k].shape, dtype, at("grad_" + k))
        f32 = lambda *s: torch.zeros(*s, device=dev)  # noqa: E731
        memory, states, grad_memory = f32(B, H, P, N), f32(B, (T + 63) // 64, H, P, N), f32(B, H, P, N)
        n = lib.grm_hip_delta_scan_workspace(B, T, H, P, N, code)
        ws = torch.zeros(n, dtype=torch.uint8, device=dev)
        p = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
        assert lib.grm_hip_delta_scan_fwd(ctypes.byref(a), p(out["hidden"]), p(memory), p(states), p(out["miss"]), p(ws), n, stream) == capi.OK
        n = lib.grm_hip_delta_scan_bwd_workspace(B, T, H, P, G, N)
        ws2 = torch.zeros(n, dtype=torch.uint8, device=dev)
        grads = [p(out["grad_" + k]) for k in ("keys", "values", "queries", "strengths", "log_decays")]
        assert lib.grm_hip_delta_scan_bwd(ctypes.byref(a), p(states), p(out["miss"]), p(x["grad_hidden"]), None, *grads, p(grad_memory),
                                          p(ws2), n, stream) == capi.OK
        torch.cuda.synchronize()
        return dict(out, memory=memory, grad_memory=grad_memory)

    want = both(())
    assert all(t.any() for t in want.values())
    for shifted in [("hidden",), ("miss",), ("grad_hidden",), ("grad_values",), ("grad_keys",), ("grad_queries",), ("keys",), ("values",),
                    ("queries",), ("strengths", "grad_strengths"), ("log_decays", "grad_log_decays"),
                    ("grad_keys", "grad_queries", "grad_values", "hidden")]:
        got = both(shifted)
        for k, t in got.items():
            assert torch.equal(t, want[k]), (shifted, k)
