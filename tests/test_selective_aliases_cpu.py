"""Results of the selective scan and the short convolution share no memory with what they were made from."""

import pytest
import torch

from rnn_with_grm_amd import cuda_ops


@pytest.mark.parametrize("T", [0, 1, 5])
def test_results_are_tensors_of_their_own(T):
    r = lambda *s: torch.randn(*s)  # noqa: E731
    memory, state, x = r(2, 2, 3, 4), r(2, 3, 6), r(2, T, 6)
    hidden, memory_out = cuda_ops.cuda_selective_scan(r(2, T, 1, 4), r(2, T, 2, 3), r(2, T, 1, 4), r(2, T, 2), -torch.ones(2), memory)
    out, state_out = cuda_ops.cuda_short_conv(x, r(6, 4), None, state)
    kept = memory.clone(), state.clone()
    memory_out.zero_(), state_out.zero_(), out.zero_(), hidden.zero_()
    assert torch.equal(memory, kept[0]) and torch.equal(state, kept[1])
    for a in (memory_out, state_out, hidden, out):
        for b in (memory, state, x):
            assert a.untyped_storage().data_ptr() != b.untyped_storage().data_ptr() or a.numel() == 0 or b.numel() == 0
