"""What the selective scan's and the short convolution's sources and entry points keep to, without a GPU."""

import ctypes
import re
from pathlib import Path

import pytest

from rnn_with_grm_amd import capi

CSRC = Path(__file__).resolve().parents[1] / "rnn_with_grm_amd" / "csrc"


def calls(text, name):
    """The argument lists of the calls of `name` in a source."""
    for m in re.finditer(name + r"\(", text):
        args, depth = [""], 0
        for ch in text[m.end():]:
            if ch == "," and depth == 0:
                args.append("")
                continue
            depth += (ch in "([{") - (ch in ")]}")
            if depth < 0:
                break
            args[-1] += ch
        yield [x.strip() for x in args]


def test_masked_loads_have_no_scalar_offset():
    """Rows past a tile's end read zeros because their offset lies outside the buffer resource.  That holds for the
    vector register's part of an offset; a scalar one need not be in the range check."""
    found = [c for p in sorted(CSRC.glob("selective*")) for c in calls(p.read_text(), r"__builtin_amdgcn_raw_buffer_load_\w+")]
    assert len(found) >= 5 and all(len(c) == 4 for c in found)
    assert [c for c in found if c[2] != "0"] == []


# ---------------------------------------------------------------------------
# Sizes that no launch can have are refused before one; nothing below reaches a device.

FAKE = 1 << 20


def scan_args(batch, seq_len=1, heads=1, value_dim=16, dtype=capi.BF16):
    row = heads * value_dim
    return ctypes.byref(capi.SelectiveArgs(
        keys=FAKE, values=FAKE, queries=FAKE, steps=FAKE, rates=FAKE, memory=FAKE, batch=batch, seq_len=seq_len, heads=heads,
        value_dim=value_dim, groups=1, key_dim=32, keys_batch_stride=32 * seq_len, keys_token_stride=32,
        values_batch_stride=row * seq_len, values_token_stride=row, queries_batch_stride=32 * seq_len,
        queries_token_stride=32, steps_batch_stride=heads * seq_len, steps_token_stride=heads, dtype=dtype, steps_dtype=dtype,
        softplus=1))


@pytest.mark.parametrize("batch,heads,value_dim,tiles", [(1 << 23, 1, 16, 1), (1 << 22, 2, 64, 1), (1 << 20, 1, 512, 8), (1 << 16, 64, 65, 2)])
def test_scans_of_too_many_workgroups(batch, heads, value_dim, tiles):
    """512 threads for each of batch * heads * value tiles: 2^32 threads, one more than a grid's dimension has."""
    lib = capi.load()
    assert batch * heads * tiles == 1 << 23
    call = lambda b, out: lib.grm_hip_selective_scan_fwd(scan_args(b, 1, heads, value_dim), out, out, None, None, 0, None)  # noqa: E731
    back = lambda b: lib.grm_hip_selective_scan_bwd(scan_args(b, 1, heads, value_dim), None, None, None, None, None, None,  # noqa: E731
                                                    None, None, None, None, None, None, 0, None)
    assert call(batch, 1 << 40) == back(batch) == capi.EUNSUPPORTED and "below 8388608" in capi.last_error()
    assert call(batch - 1, None) == back(batch - 1) == capi.EINVAL  # the next refusal: no outputs


def test_steps_of_too_many_workgroups():
    lib = capi.load()
    step = lambda b, **kw: lib.grm_hip_selective_step(scan_args(b, **kw), None, None, None)  # noqa: E731
    assert step(1 << 24) == step(1 << 22, heads=4, value_dim=512) == capi.EUNSUPPORTED
    assert step((1 << 24) - 1) == step((1 << 22) - 1, heads=4, value_dim=512) == capi.EINVAL


@pytest.mark.parametrize("dtype,block", [(capi.BF16, 128), (capi.F32, 64)])
def test_gradients_of_too_many_blocks(dtype, block):
    lib = capi.load()
    back = lambda T: lib.grm_hip_selective_scan_bwd(scan_args(16, T, dtype=dtype), FAKE, FAKE, None, FAKE, FAKE, FAKE, FAKE,  # noqa: E731
                                                    FAKE, FAKE, None, None, FAKE, 1 << 62, None)
    assert back(block << 19) == capi.EUNSUPPORTED  # 2^23 workgroups of 512 threads


def test_convolution_weights_of_too_many_channels():
    C = (1 << 29) // 5
    assert -(-C * 5 // 64) == 1 << 23  # workgroups of 512 threads
    back = capi.load().grm_hip_short_conv_bwd(FAKE, FAKE, None, None, None, FAKE, None, FAKE, FAKE, None, None, FAKE, 1 << 62, 1, 1, C,
                                              4, C, C, capi.BF16, capi.BF16, 0, None)
    assert back == capi.EUNSUPPORTED


@pytest.mark.parametrize("B,T,C", [(1 << 62, 1, 4), (4, 1 << 62, 4), (4, 1, 1 << 62), (1 << 30, 1 << 30, 16), ((1 << 63) - 1, 8, 8),
                                   (1 << 40, 1 << 12, 1), (2, (1 << 63) - 1, 2)])
def test_convolutions_whose_sizes_pass_63_bits(B, T, C):
    """Their products would wrap round to a small launch."""
    lib = capi.load()
    assert lib.grm_hip_short_conv_fwd(FAKE, FAKE, None, None, None, FAKE, 2 * FAKE, B, T, C, 4, T * C % (1 << 62), C, 0, 0, 0, None) == capi.EUNSUPPORTED
    assert lib.grm_hip_short_conv_bwd_workspace(B, T, C, 4, 0) == 0
    assert lib.grm_hip_short_conv_bwd(FAKE, FAKE, None, None, None, FAKE, None, FAKE, FAKE, None, None, FAKE, 1 << 62, B, T, C, 4,
                                      T * C % (1 << 62), C, 0, 0, 0, None) == capi.EUNSUPPORTED
    if T == 1:
        assert lib.grm_hip_short_conv_step(FAKE, FAKE, None, FAKE, FAKE, FAKE, B, C, 4, C, 0, 0, 0, None) == capi.EUNSUPPORTED
