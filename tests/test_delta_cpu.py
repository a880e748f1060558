"""The PyTorch forms of the delta rule and the group norm, and the refusals of their entry points and of the C ABI,
none of which needs a GPU."""

import ctypes

import pytest
import torch

import delta_oracle as oracle
from rnn_with_grm_amd import capi, cuda_ops

NAMES = oracle.NAMES


def inputs(B, T, H, P, G, N, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    unit = lambda *s: torch.nn.functional.normalize(r(*s), dim=-1)  # noqa: E731
    return [unit(B, T, G, N).to(dtype), r(B, T, H, P).to(dtype), unit(B, T, G, N).to(dtype),
            torch.sigmoid(r(B, T, H)).to(dtype), -torch.exp(r(B, T, H) - 1).to(dtype), r(B, H, P, N).to(dtype)]


@pytest.mark.parametrize("lengths", [None, (9, 4), (0, 99)])
def test_scan_is_the_definition(lengths):
    x = inputs(2, 9, 4, 3, 2, 5, torch.float64)
    n = None if lengths is None else torch.tensor(lengths)
    leaves = [t.requires_grad_() for t in x]
    got = cuda_ops.cuda_delta_scan(*leaves, lengths=n)
    want = oracle.delta_scan(*leaves, n)
    for a, b in zip(got, want):
        torch.testing.assert_close(a, b, rtol=1e-12, atol=1e-12)
    w = [torch.randn_like(t) for t in want]
    for a, b in zip(torch.autograd.grad(got, leaves, w), torch.autograd.grad(want, leaves, w)):
        torch.testing.assert_close(a, b, rtol=1e-10, atol=1e-12)


def test_gradients_against_differences():
    leaves = [t.requires_grad_() for t in inputs(1, 4, 2, 2, 1, 3, torch.float64)]
    assert torch.autograd.gradcheck(lambda *a: cuda_ops.cuda_delta_scan(*a, lengths=torch.tensor([3])), leaves)
    x = torch.randn(3, 6, dtype=torch.float64, requires_grad=True)
    w, b, z = (torch.randn(s, dtype=torch.float64, requires_grad=True) for s in ((6,), (6,), (3, 6)))
    for center in (True, False):
        assert torch.autograd.gradcheck(lambda *a: cuda_ops.cuda_group_norm(a[0], 2, *a[1:], activation="silu", center=center), (x, w, b, z))
        assert torch.autograd.gradcheck(lambda *a: cuda_ops.cuda_group_norm(a[0], 3, *a[1:], activation="silu", center=center), (x, w, b))


def test_steps_follow_the_scan():
    x = inputs(2, 3, 2, 4, 1, 4, torch.float32)
    hidden, memory = cuda_ops.cuda_delta_scan(*x)
    state = x[5].clone()
    for t in range(3):
        out, same = cuda_ops.cuda_delta_step(*(v[:, t] for v in x[:5]), state, memory_out=state)
        assert same is state
        torch.testing.assert_close(out, hidden[:, t])
    torch.testing.assert_close(state, memory)
    none = cuda_ops.cuda_delta_step(*(v[:, 0] for v in x[:4]), None, x[5])
    zero = cuda_ops.cuda_delta_step(*(v[:, 0] for v in x[:4]), torch.zeros(2, 2), x[5])
    assert torch.equal(none[0], zero[0]) and torch.equal(none[1], zero[1])
    empty = cuda_ops.cuda_delta_scan(*(v[:, :0] for v in x[:5]), x[5])
    assert empty[0].shape == (2, 0, 2, 4) and torch.equal(empty[1], x[5]) and empty[1] is not x[5]


def test_no_earlier_token_sees_an_infinity():
    x = inputs(1, 6, 1, 3, 1, 4, torch.float32)
    want = cuda_ops.cuda_delta_scan(*x)[0]
    for i in range(5):
        y = [t.clone() for t in x]
        y[i][(0, 3) + (0,) * (y[i].ndim - 2)] = float("inf")
        assert torch.equal(cuda_ops.cuda_delta_scan(*y)[0][:, :3], want[:, :3])


@pytest.mark.parametrize("center", [True, False])
def test_norm_is_the_definition(center):
    g = torch.Generator().manual_seed(1)
    x, z = (torch.randn(5, 12, generator=g, dtype=torch.float64) for _ in range(2))
    w, b = (torch.randn(12, generator=g, dtype=torch.float64) for _ in range(2))
    for gate in (None, z):
        for act in (None, "silu"):
            got = cuda_ops.cuda_group_norm(x, 3, w, b, gate, activation=act, center=center)
            torch.testing.assert_close(got, oracle.group_norm(x, 3, w, b, gate, act is not None, center), rtol=1e-12, atol=1e-12)
    assert cuda_ops.cuda_group_norm(x.bfloat16().view(1, 5, 12), 3).shape == (1, 5, 12)
    torch.testing.assert_close(cuda_ops.cuda_group_norm(x, 3, w, b), torch.nn.functional.group_norm(x, 3, w, b))


def test_refusals():
    x = inputs(2, 3, 4, 3, 2, 5, torch.float32)
    for i, bad, match in [(0, x[0][:, :2], "agree"), (1, x[1].half(), "share a type"), (2, x[2][..., :4], "agree"),
                          (3, x[3][..., :2], "agree"), (3, x[3].half(), "float32"), (4, x[4][:1], "agree"), (5, x[5][:1], "memory"),
                          (0, x[0][:, :, 0], "must be"), (0, x[0].repeat(1, 1, 2, 1)[:, :, :3], "agree")]:
        y = list(x)
        y[i] = bad
        with pytest.raises(ValueError, match=match):
            cuda_ops.cuda_delta_scan(*y)
    with pytest.raises(ValueError, match="lengths"):
        cuda_ops.cuda_delta_scan(*x, lengths=torch.zeros(3, dtype=torch.long))
    with pytest.raises(ValueError, match="must be"):
        cuda_ops.cuda_delta_step(*x)
    one = [t[:, 0] for t in x[:5]]
    with pytest.raises(ValueError, match="match"):
        cuda_ops.cuda_delta_step(*one, x[5], memory_out=x[5][:1])
    with pytest.raises(ValueError, match="gradients"):
        cuda_ops.cuda_delta_step(*one, x[5].clone().requires_grad_(), memory_out=x[5])
    v = torch.zeros(2, 12)
    for kw, match in [(dict(groups=5), "multiple"), (dict(weight=v[0, :4]), "weight"), (dict(gate=v[:1]), "gate"), (dict(eps=-1.0), "eps"),
                      (dict(activation="relu"), "activation"), (dict(weight=v[0], bias=v[0].half()), "bias")]:
        kw = dict(dict(groups=3), **kw)
        with pytest.raises(ValueError, match=match):
            cuda_ops.cuda_group_norm(v, kw.pop("groups"), **kw)


def fake(n=16):
    return ctypes.c_void_p(n)  # never dereferenced: validation fails first


def delta_args(**kw):
    a = capi.DeltaArgs()
    for f in ("keys", "values", "queries", "strengths", "log_decays"):
        setattr(a, f, 16)
    sizes = dict(batch=2, seq_len=4, heads=4, value_dim=8, groups=2, key_dim=8, keys_batch_stride=64, keys_token_stride=16,
                 values_batch_stride=128, values_token_stride=32, queries_batch_stride=64, queries_token_stride=16,
                 strengths_batch_stride=16, strengths_token_stride=4, decays_batch_stride=16, decays_token_stride=4,
                 dtype=capi.BF16, strengths_dtype=capi.BF16, decays_dtype=capi.F32)
    for k, v in dict(sizes, **kw).items():
        setattr(a, k, v)
    return a


BAD = [
    (dict(batch=-1), capi.EINVAL), (dict(heads=0), capi.EINVAL), (dict(heads=3), capi.EINVAL), (dict(key_dim=129), capi.EUNSUPPORTED),
    (dict(dtype=7), capi.EUNSUPPORTED), (dict(strengths_dtype=capi.F16), capi.EUNSUPPORTED), (dict(decays_dtype=5), capi.EUNSUPPORTED),
    (dict(seq_len=2 ** 31), capi.EUNSUPPORTED), (dict(heads=2 ** 22, groups=2 ** 22), capi.EUNSUPPORTED),
    (dict(value_dim=2 ** 62), capi.EUNSUPPORTED), (dict(batch=2 ** 62), capi.EUNSUPPORTED), (dict(keys_token_stride=15), capi.EINVAL),
    (dict(values_token_stride=2 ** 22), capi.EUNSUPPORTED), (dict(batch=2 ** 21, heads=4), capi.EUNSUPPORTED), (dict(seq_len=2 ** 27 + 1, batch=1), capi.EUNSUPPORTED),
    (dict(keys=None), capi.EINVAL), (dict(strengths=None), capi.EINVAL), (dict(memory=20), capi.EINVAL),
]


@pytest.mark.parametrize("kw,code", BAD)
def test_c_entry_points_refuse(kw, code):
    a = delta_args(**kw)
    lib = capi.load()
    assert lib.grm_hip_delta_scan_fwd(ctypes.byref(a), fake(), fake(32), None, None, fake(), 1 << 40, None) == code
    assert capi.last_error()
    assert lib.grm_hip_delta_scan_bwd(ctypes.byref(a), *[fake()] * 11, 1 << 40, None) == code
    b = delta_args(**dict(kw, seq_len=kw.get("seq_len", 1)))
    if kw not in (dict(keys_token_stride=15), dict(batch=2 ** 21, heads=4)):  # (one token has no stride, and a smaller grid)
        assert lib.grm_hip_delta_step(ctypes.byref(b), fake(), fake(32), None) in (code, capi.EINVAL)


def test_c_entry_points_need_their_buffers():
    lib = capi.load()
    a = delta_args()
    ref = ctypes.byref(a)
    wsb = lib.grm_hip_delta_scan_workspace(2, 4, 4, 8, 8, capi.BF16)
    assert wsb > 0 and lib.grm_hip_delta_scan_workspace(2, 0, 4, 8, 8, capi.BF16) == 0
    for args in [(None, fake(32), None, None, fake(), wsb), (fake(), None, None, None, fake(), wsb), (fake(), fake(32), None, None, None, wsb),
                 (fake(), fake(32), None, None, fake(), wsb - 1), (fake(), fake(32), None, None, fake(8), wsb), (fake(), fake(40), None, None, fake(), wsb),
                 (fake(), fake(32), fake(), None, fake(), wsb), (fake(), fake(32), None, fake(), fake(), wsb)]:
        assert lib.grm_hip_delta_scan_fwd(ref, *args, None) == capi.EINVAL
    a.memory = 64
    assert lib.grm_hip_delta_scan_fwd(ref, fake(), fake(128), None, None, fake(), wsb, None) == capi.EINVAL
    assert b"overlap" in lib.grm_hip_last_error()
    bws = lib.grm_hip_delta_scan_bwd_workspace(2, 4, 4, 8, 2, 8)
    good = [fake()] * 11
    for i in (0, 1, 2, 4, 5, 6, 7, 9, 10):
        args = list(good)
        args[i] = None
        assert lib.grm_hip_delta_scan_bwd(ref, *args, bws, None) == capi.EINVAL, i
    assert lib.grm_hip_delta_scan_bwd(ref, *good, bws - 1, None) == capi.EINVAL
    assert lib.grm_hip_delta_step(ref, fake(), fake(32), None) == capi.EINVAL  # (more than one token)
    none = delta_args(batch=0)
    assert lib.grm_hip_delta_scan_fwd(ctypes.byref(none), None, None, None, None, None, 0, None) == capi.OK
    assert lib.grm_hip_delta_scan_fwd(None, None, None, None, None, None, 0, None) == capi.EINVAL


@pytest.mark.parametrize("kw,code", [
    (dict(rows=-1), capi.EINVAL), (dict(groups=5), capi.EINVAL), (dict(channels=0), capi.EINVAL), (dict(dtype=3), capi.EUNSUPPORTED),
    (dict(weight_dtype=capi.F16), capi.EUNSUPPORTED), (dict(channels=8194, groups=2), capi.EUNSUPPORTED),
    (dict(channels=2 ** 22, groups=2 ** 21), capi.EUNSUPPORTED), (dict(eps=-1.0), capi.EINVAL), (dict(eps=float("nan")), capi.EINVAL),
    (dict(x_stride=11), capi.EUNSUPPORTED), (dict(rows=2 ** 32), capi.EUNSUPPORTED), (dict(x=None), capi.EINVAL), (dict(out=None), capi.EINVAL)])
def test_norm_entry_points_refuse(kw, code):
    a = dict(rows=4, channels=12, groups=3, x_stride=12, gate_stride=12, dtype=capi.BF16, weight_dtype=capi.BF16, eps=1e-5, x=fake(), out=fake())
    a.update(kw)
    lib = capi.load()
    rest = (a["rows"], a["channels"], a["groups"], a["x_stride"], a["gate_stride"], a["dtype"], a["weight_dtype"], 1, 1, a["eps"], None)
    assert lib.grm_hip_group_norm_fwd(a["x"], fake(), fake(), fake(), a["out"], *rest) == code
    assert lib.grm_hip_group_norm_bwd(a["x"], fake(), fake(), fake(), fake(), a["out"], fake(), fake(), fake(), fake(), 1 << 40, *rest) == code
    assert lib.grm_hip_group_norm_fwd(None, None, None, None, None, 0, 12, 3, 12, 12, capi.F32, capi.F32, 0, 1, 1e-5, None) == capi.OK
