"""Calls that need the keys' weights refuse to go without them, without a GPU."""
import pytest
import torch

import dashmag_amd as dm
from dashmag_amd.contract import Unsupported


def test_weights_that_are_missing():
    q, k, table = torch.zeros(2, 4, 64), torch.zeros(3, 16, 2, 64), torch.zeros(2, 2, dtype=torch.int32)
    with pytest.raises(Unsupported, match="^attention_paged_with_weights: the weights are missing"):
        dm.attention_paged_with_weights(q, k, k, table, [3, 4], None)
    lengths, counts = (torch.zeros(n, dtype=torch.int32) for n in (2, 3))
    with pytest.raises(Unsupported, match="^cache_evict: the weights are missing"):
        dm.cache_evict([k], None, table, lengths, counts, [1, 1])
