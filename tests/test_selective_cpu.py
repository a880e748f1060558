"""The selective scan and the short convolution without a GPU: the PyTorch forms against the float64
definitions (results, gradients, refusals), and the C entry points' checks, which come before any launch."""

import ctypes

import pytest
import torch

import selective_oracle as oracle
from rnn_with_grm_amd import capi, cuda_ops


def scan_inputs(B, T, H, P, G, N, dtype=torch.float64, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=dtype)  # noqa: E731
    return dict(keys=r(B, T, G, N), values=r(B, T, H, P), queries=r(B, T, G, N), steps=r(B, T, H) - 2,
                rates=-torch.exp(r(H)), memory=r(B, H, P, N), skip=r(H), step_bias=r(H) - 1)


NAMES = ("keys", "values", "queries", "steps", "rates", "memory", "skip", "step_bias")


def scan(x, lengths=None, softplus=True):
    return cuda_ops.cuda_selective_scan(x["keys"], x["values"], x["queries"], x["steps"], x["rates"], x["memory"],
                                        skip=x["skip"], step_bias=x["step_bias"], softplus=softplus, lengths=lengths)


@pytest.mark.parametrize("T,lengths", [(1, None), (70, None), (130, (130, 65)), (9, (0, 100)), (5, (-1, 3)), (0, None)])
def test_scan_and_its_gradients(T, lengths):
    """float64 throughout: a few hundred roundings of 2^-53 against sums of order 10."""
    x = {k: v.requires_grad_() for k, v in scan_inputs(2, T, 4, 5, 2, 6).items()}
    n = None if lengths is None else torch.tensor(lengths)
    out = scan(x, n)
    ref_in = {k: v.detach().clone().requires_grad_() for k, v in x.items()}
    ref = oracle.selective_scan(*(ref_in[k] for k in NAMES), n, True)
    for a, b in zip(out, ref):
        torch.testing.assert_close(a, b, rtol=1e-10, atol=1e-10)
    ups = [torch.randn(o.shape, dtype=torch.float64) for o in ref]
    got = torch.autograd.grad(out, [x[k] for k in NAMES], ups, allow_unused=True)
    want = torch.autograd.grad(ref, [ref_in[k] for k in NAMES], ups, allow_unused=True)
    for k, a, b in zip(NAMES, got, want):
        a, b = (torch.zeros_like(x[k]) if v is None else v for v in (a, b))
        torch.testing.assert_close(a, b, rtol=1e-9, atol=1e-9, msg=lambda m, k=k: f"{k}: {m}")


def test_scan_continues_and_steps():
    """A prompt in two calls, and token by token, as in one."""
    x = scan_inputs(2, 12, 4, 5, 2, 6)
    hidden, memory = scan(x)
    cut = lambda lo, hi, m: dict(x, memory=m, **{k: x[k][:, lo:hi] for k in ("keys", "values", "queries", "steps")})  # noqa: E731
    a, m = scan(cut(0, 7, x["memory"]))
    b, m = scan(cut(7, 12, m))
    torch.testing.assert_close(torch.cat([a, b], 1), hidden, rtol=1e-10, atol=1e-10)
    torch.testing.assert_close(m, memory, rtol=1e-10, atol=1e-10)
    kept = x["memory"].clone()
    for t in range(12):
        h, out = cuda_ops.cuda_selective_step(x["keys"][:, t], x["values"][:, t], x["queries"][:, t], x["steps"][:, t],
                                              x["rates"], kept, skip=x["skip"], step_bias=x["step_bias"], softplus=True,
                                              memory_out=kept)
        assert out is kept
        torch.testing.assert_close(h, hidden[:, t], rtol=1e-10, atol=1e-10)
    torch.testing.assert_close(kept, memory, rtol=1e-10, atol=1e-10)


@pytest.mark.parametrize("T,W,silu,lengths", [(1, 4, True, None), (20, 3, False, None), (9, 2, True, (9, 0)), (3, 4, True, (50, -2)),
                                              (0, 4, True, None)])
def test_convolution_and_its_gradients(T, W, silu, lengths):
    g = torch.Generator().manual_seed(T)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).requires_grad_()  # noqa: E731
    x = (r(2, T, 7), r(7, W), r(7), r(2, W - 1, 7))
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32)
    out = cuda_ops.cuda_short_conv(*x, activation="silu" if silu else None, lengths=n)
    ref = oracle.short_conv(*x, n, silu)
    for a, b in zip(out, ref):
        torch.testing.assert_close(a, b, rtol=1e-12, atol=1e-12)
    ups = [torch.randn(o.shape, dtype=torch.float64) for o in ref]
    got = torch.autograd.grad(out, x, ups, allow_unused=True)
    want = torch.autograd.grad(ref, x, ups, allow_unused=True)
    for a, b, v in zip(got, want, x):
        a, b = (torch.zeros_like(v) if u is None else u for u in (a, b))
        torch.testing.assert_close(a, b, rtol=1e-11, atol=1e-11)


def test_convolution_steps():
    g = torch.Generator().manual_seed(1)
    x, w, b, st = (torch.randn(*s, generator=g) for s in ((2, 6, 5), (5, 4), (5,), (2, 3, 5)))
    out, state = cuda_ops.cuda_short_conv(x, w, b, st, activation="silu")
    kept = st.clone()
    for t in range(6):
        y, same = cuda_ops.cuda_short_conv_step(x[:, t], kept, w, b, activation="silu", state_out=kept)
        assert same is kept
        torch.testing.assert_close(y, out[:, t])
    assert torch.equal(kept, state)


def test_refusals():
    x = scan_inputs(2, 5, 4, 3, 2, 6, torch.float32)
    bad = (dict(keys=x["keys"][:, :3]), dict(keys=x["keys"][..., :4]), dict(values=x["values"][:, :, :3]),
           dict(values=x["values"].half()), dict(steps=x["steps"].double()), dict(rates=x["rates"][:2]),
           dict(memory=x["memory"][:1]), dict(skip=x["skip"][:1]), dict(step_bias=x["step_bias"][:, None]),
           dict(keys=torch.zeros(2, 5, 2, 129), queries=torch.zeros(2, 5, 2, 129), memory=None),
           dict(keys=x["keys"][:, :, :0], queries=x["queries"][:, :, :0]))
    for more in bad:
        with pytest.raises(ValueError):
            scan({**x, **more})
    for lengths in (torch.zeros(3, dtype=torch.long), torch.zeros(2)):
        with pytest.raises(ValueError):
            scan(x, lengths)
    c, w = torch.zeros(2, 5, 6), torch.zeros(6, 4)
    for call in (lambda: cuda_ops.cuda_short_conv(c, w[:, :1]), lambda: cuda_ops.cuda_short_conv(c, torch.zeros(6, 5)),
                 lambda: cuda_ops.cuda_short_conv(c, w[:4]), lambda: cuda_ops.cuda_short_conv(c, w, torch.zeros(3)),
                 lambda: cuda_ops.cuda_short_conv(c, w, state=torch.zeros(2, 2, 6)),
                 lambda: cuda_ops.cuda_short_conv(c, w, activation="gelu"),
                 lambda: cuda_ops.cuda_short_conv_step(c, torch.zeros(2, 3, 6), w),
                 lambda: cuda_ops.cuda_short_conv_step(c[:, 0], torch.zeros(2, 3, 6), w, state_out=torch.zeros(2, 3, 5)),
                 lambda: cuda_ops.cuda_selective_step(x["keys"], x["values"], x["queries"], x["steps"], x["rates"],
                                                      x["memory"])):
        with pytest.raises(ValueError):
            call()


# ---------------------------------------------------------------------------
# C entry points: everything below is refused before a launch; no pointer is followed.

FAKE = 1 << 20  # 16-byte aligned


def selective_args(**kw):
    a = dict(keys=FAKE, values=FAKE, queries=FAKE, steps=FAKE, rates=FAKE, memory=FAKE, batch=2, seq_len=8, heads=4,
             value_dim=16, groups=2, key_dim=32, keys_batch_stride=512, keys_token_stride=64, values_batch_stride=512,
             values_token_stride=64, queries_batch_stride=512, queries_token_stride=64, steps_batch_stride=32,
             steps_token_stride=4, dtype=capi.BF16, steps_dtype=capi.BF16, softplus=1)
    a.update(kw)
    return capi.SelectiveArgs(**a)


BAD = [
    (dict(batch=-1), capi.EINVAL), (dict(seq_len=-1), capi.EINVAL), (dict(heads=0), capi.EINVAL),
    (dict(heads=3), capi.EINVAL), (dict(key_dim=0), capi.EINVAL), (dict(key_dim=129), capi.EUNSUPPORTED),
    (dict(dtype=3), capi.EUNSUPPORTED), (dict(steps_dtype=capi.F16), capi.EUNSUPPORTED), (dict(keys=None), capi.EINVAL),
    (dict(rates=None), capi.EINVAL), (dict(memory=FAKE + 4), capi.EINVAL), (dict(keys_token_stride=63), capi.EINVAL),
    (dict(values_token_stride=1 << 22), capi.EUNSUPPORTED), (dict(seq_len=1 << 31), capi.EUNSUPPORTED),
    (dict(batch=1 << 24), capi.EUNSUPPORTED), (dict(batch=1 << 62), capi.EUNSUPPORTED),
    (dict(heads=1 << 62, groups=1), capi.EUNSUPPORTED), (dict(value_dim=1 << 62), capi.EUNSUPPORTED),
]


@pytest.mark.parametrize("kw,code", BAD)
def test_c_scan_refuses(kw, code):
    lib = capi.load()
    out = 2 * FAKE
    assert lib.grm_hip_selective_scan_fwd(ctypes.byref(selective_args(**kw)), out, out, None, None, 0, None) == code
    assert capi.last_error()
    assert lib.grm_hip_selective_scan_bwd(ctypes.byref(selective_args(**kw)), out, out, None, out, out, out, out, out, out, None,
                                          None, out, 1 << 40, None) == code


def test_c_scan_refuses_outputs_and_workspaces():
    lib = capi.load()
    out = 2 * FAKE
    call = lambda a, hidden, memory, ws, n: lib.grm_hip_selective_scan_fwd(ctypes.byref(a), hidden, memory, None, ws, n, None)  # noqa: E731
    assert call(selective_args(), None, out, None, 0) == capi.EINVAL
    assert call(selective_args(), out, None, None, 0) == capi.EINVAL
    assert call(selective_args(), out, out + 4, None, 0) == capi.EINVAL
    assert call(selective_args(), out, FAKE, None, 0) == capi.EINVAL          # the final state over the first
    long = selective_args(batch=1, seq_len=4096, heads=2)
    need = lib.grm_hip_selective_scan_workspace(1, 4096, 2, 16, 32, capi.BF16)
    assert need > 0                                                            # few heads: time parts
    assert call(long, out, out, None, need) == capi.EINVAL
    assert call(long, out, out, 4 * FAKE, need - 1) == capi.EINVAL
    assert lib.grm_hip_selective_scan_workspace(64, 4096, 8, 16, 32, capi.BF16) == 0
    back = lambda a, ws, n, states=out: lib.grm_hip_selective_scan_bwd(  # noqa: E731
        ctypes.byref(a), states, out, None, out, out, out, out, out, out, None, None, ws, n, None)
    need = lib.grm_hip_selective_scan_bwd_workspace(2, 8, 4, 16, 2, 32, capi.BF16)
    assert need > 0 and back(selective_args(), 4 * FAKE, need - 1) == capi.EINVAL
    assert back(selective_args(), None, need) == capi.EINVAL and back(selective_args(), 4 * FAKE, need, None) == capi.EINVAL
    step = lambda a, hidden, memory: lib.grm_hip_selective_step(ctypes.byref(a), hidden, memory, None)  # noqa: E731
    assert step(selective_args(), out, out) == capi.EINVAL                     # eight tokens
    assert step(selective_args(seq_len=1, lengths=FAKE), out, out) == capi.EINVAL
    assert step(selective_args(seq_len=1, memory=None), out, out) == capi.EINVAL
    assert step(selective_args(seq_len=1), out, FAKE + 16) == capi.EINVAL      # half over the old state


def test_c_convolution_refuses():
    lib = capi.load()
    F, O = FAKE, 2 * FAKE

    def fwd(x=F, w=F, state=None, out=O, state_out=3 * FAKE, B=2, T=8, C=16, W=4, dtype=capi.F32, wdtype=capi.F32):
        return lib.grm_hip_short_conv_fwd(x, w, None, state, None, out, state_out, B, T, C, W, T * C, C, dtype, wdtype, 1, None)

    assert fwd(B=-1) == fwd(T=-1) == fwd(C=0) == capi.EINVAL
    assert fwd(W=1) == fwd(W=5) == fwd(dtype=9) == fwd(dtype=capi.F32, wdtype=capi.F16) == capi.EUNSUPPORTED
    assert fwd(x=None) == fwd(w=None) == fwd(out=None) == fwd(state_out=None) == fwd(state=3 * FAKE) == capi.EINVAL
    assert fwd(B=1 << 20, T=1 << 20, C=1 << 10) == capi.EUNSUPPORTED
    need = lib.grm_hip_short_conv_bwd_workspace(2, 8, 16, 4, capi.F32)
    back = lambda ws, n, dw=O: lib.grm_hip_short_conv_bwd(F, F, None, None, None, O, None, O, dw, None, None, ws, n, 2, 8, 16, 4,  # noqa: E731
                                                          128, 16, capi.F32, capi.F32, 1, None)
    assert need > 0 and back(4 * FAKE, need - 1) == back(None, need) == back(4 * FAKE, need, None) == capi.EINVAL
    step = lambda state, state_out: lib.grm_hip_short_conv_step(F, F, None, state, O, state_out, 2, 16, 4, 16, capi.F32, capi.F32, 1, None)  # noqa: E731
    assert step(None, O) == step(F, None) == step(F, F + 64) == capi.EINVAL


def test_empty_batches_launch_nothing():
    lib = capi.load()
    before = capi.launch_count()
    assert lib.grm_hip_selective_scan_fwd(ctypes.byref(selective_args(batch=0)), None, None, None, None, 0, None) == capi.OK
    assert lib.grm_hip_selective_step(ctypes.byref(selective_args(batch=0, seq_len=1)), None, None, None) == capi.OK
    assert lib.grm_hip_short_conv_fwd(None, None, None, None, None, None, None, 0, 8, 16, 4, 128, 16, 0, 0, 1, None) == capi.OK
    assert capi.launch_count() == before
