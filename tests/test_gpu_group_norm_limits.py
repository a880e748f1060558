"""Sizes that the group norm does not take are refused before anything of these sizes is allocated (the rows here are broadcast
from a single element, and would be laid out anew)."""

import pytest
import torch

from rnn_with_grm_amd import cuda_ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,channels,groups,match", [(4096, 2 ** 22, 2 ** 21, r"2\^21 channels"), (2 ** 31 + 1, 8, 1, r"2\^31 rows")])
def test_refused_before_any_allocation(dev, rows, channels, groups, match):
    one = torch.zeros(1, dtype=torch.bfloat16, device=dev)
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.max_memory_allocated()
    with pytest.raises(RuntimeError, match=match):
        cuda_ops.cuda_group_norm(one.expand(rows, channels), groups)
    assert torch.cuda.max_memory_allocated() <= before + 4096
