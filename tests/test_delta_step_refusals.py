"""The single token's C entry point of the delta rule: each refusal by its own code.  Nothing here needs a GPU: every call is refused.

All buffers are given (16-byte aligned, apart from each other), so that a call fails only for what its row names."""

import ctypes

import pytest

from rnn_with_grm_amd import capi

GOOD = dict(keys=0x1000, values=0x2000, queries=0x3000, strengths=0x4000, log_decays=0x5000, memory=0x100000, lengths=None, batch=2, seq_len=1,
            heads=4, value_dim=8, groups=2, key_dim=8, keys_batch_stride=16, keys_token_stride=16, values_batch_stride=32,
            values_token_stride=32, queries_batch_stride=16, queries_token_stride=16, strengths_batch_stride=4, strengths_token_stride=4,
            decays_batch_stride=4, decays_token_stride=4, dtype=capi.BF16, strengths_dtype=capi.BF16, decays_dtype=capi.F32)
STATE = 2 * 4 * 8 * 8 * 4  # bytes

REFUSED = [
    (dict(batch=-1), capi.EINVAL, b">= 0"), (dict(seq_len=-1), capi.EINVAL, b">= 0"), (dict(heads=0), capi.EINVAL, b">= 1"),
    (dict(value_dim=0), capi.EINVAL, b">= 1"), (dict(groups=0), capi.EINVAL, b">= 1"), (dict(key_dim=0), capi.EINVAL, b">= 1"),
    (dict(heads=3), capi.EINVAL, b"multiple"), (dict(dtype=7), capi.EUNSUPPORTED, b"must be float32"), (dict(dtype=-1), capi.EUNSUPPORTED, b"must be float32"),
    (dict(strengths_dtype=capi.F16), capi.EUNSUPPORTED, b"the same or float32"), (dict(decays_dtype=5), capi.EUNSUPPORTED, b"the same or float32"),
    (dict(key_dim=129), capi.EUNSUPPORTED, b"key_dim"), (dict(heads=2 ** 22, groups=2 ** 22), capi.EUNSUPPORTED, b"2^21"),
    (dict(value_dim=2 ** 62), capi.EUNSUPPORTED, b"2^21"), (dict(heads=2 ** 11, value_dim=2 ** 11), capi.EUNSUPPORTED, b"2^21"),
    (dict(batch=2 ** 62), capi.EUNSUPPORTED, b"2^24"), (dict(batch=2 ** 22), capi.EUNSUPPORTED, b"2^24"),
    (dict(keys_token_stride=2 ** 22), capi.EUNSUPPORTED, b"2^21"), (dict(values_token_stride=-1), capi.EUNSUPPORTED, b"2^21"),
    (dict(queries_token_stride=2 ** 40), capi.EUNSUPPORTED, b"2^21"), (dict(seq_len=2), capi.EINVAL, b"seq_len must be 1"),
    (dict(seq_len=0), capi.EINVAL, b"seq_len must be 1"), (dict(seq_len=2 ** 31), capi.EUNSUPPORTED, b"2^30"),
    (dict(lengths=0x6000), capi.EINVAL, b"without lengths"), (dict(keys=None), capi.EINVAL, b"required"), (dict(values=None), capi.EINVAL, b"required"),
    (dict(queries=None), capi.EINVAL, b"required"), (dict(strengths=None), capi.EINVAL, b"required"), (dict(memory=None), capi.EINVAL, b"memory, hidden"),
    (dict(memory=0x100008), capi.EINVAL, b"aligned"), (dict(hidden=None), capi.EINVAL, b"memory, hidden"), (dict(memory_out=None), capi.EINVAL, b"memory, hidden"),
    (dict(memory_out=0x200004), capi.EINVAL, b"aligned"), (dict(memory_out=0x100000 + STATE - 16), capi.EINVAL, b"overlap"),
    (dict(memory_out=0x100000 - 16), capi.EINVAL, b"overlap"),
]


@pytest.mark.parametrize("change,code,says", REFUSED)
def test_refused_with_its_own_code(change, code, says):
    values = dict(GOOD, hidden=0x7000, memory_out=0x200000)
    values.update(change)
    a = capi.DeltaArgs()
    for k, v in values.items():
        if k not in ("hidden", "memory_out"):
            setattr(a, k, v)
    lib = capi.load()
    got = lib.grm_hip_delta_step(ctypes.byref(a), *(None if values[k] is None else ctypes.c_void_p(values[k]) for k in ("hidden", "memory_out")), None)
    assert got == code and says in lib.grm_hip_last_error(), (got, lib.grm_hip_last_error())


def test_no_arguments():
    assert capi.load().grm_hip_delta_step(None, ctypes.c_void_p(16), ctypes.c_void_p(32), None) == capi.EINVAL
