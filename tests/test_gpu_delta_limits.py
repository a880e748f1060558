"""Sizes that the delta rule's launches do not take are refused as such, before anything of these sizes is allocated.

The inputs are broadcast from single elements, so that they take no memory; what a call of their sizes would allocate passes
what a card holds."""

import pytest
import torch

from rnn_with_grm_amd import cuda_ops

pytestmark = pytest.mark.gpu


def call(dev, B, T, H, P, G, N):
    one = torch.zeros(1, dtype=torch.bfloat16, device=dev)
    return cuda_ops.cuda_delta_scan(one.expand(B, T, G, N), one.expand(B, T, H, P), one.expand(B, T, G, N), one.expand(B, T, H))


@pytest.mark.parametrize("sizes,match", [
    ((1, 2 ** 30, 1, 64, 1, 64), r"ceil\(seq_len / 64\) must be below 2\^23"), ((1, 2 ** 31, 1, 64, 1, 64), r"at most 2\^30"),
    ((2 ** 23, 100, 2, 64, 1, 128), r"below 2\^23"), ((4, 1000, 1, 2 ** 22, 1, 128), r"2\^21 elements")])
def test_refused_before_any_allocation(dev, sizes, match):
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.max_memory_allocated()
    with pytest.raises(RuntimeError, match=match):
        call(dev, *sizes)
    assert torch.cuda.max_memory_allocated() <= before + 4096  # (the single element)


def test_refused_tokens(dev):
    one = torch.zeros(1, dtype=torch.bfloat16, device=dev)
    memory = torch.zeros(1, device=dev).expand(2 ** 24, 1, 64, 128)
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.max_memory_allocated()
    with pytest.raises(RuntimeError, match=r"batch \* heads must be below 2\^24"):
        cuda_ops.cuda_delta_step(one.expand(2 ** 24, 1, 128), one.expand(2 ** 24, 1, 64), one.expand(2 ** 24, 1, 128),
                                 one.expand(2 ** 24, 1), None, memory)
    assert torch.cuda.max_memory_allocated() <= before + 4096
