"""The Python operators' host side without a GPU: exceptions of the caller's own objects come through as they are."""
import pytest
import torch

import hyperattention_b200 as ha


def test_return_keys_that_is_no_truth_value():
    class Neither:
        def __bool__(self):
            raise ValueError('neither')

    c = ha.PagedCache.allocate(3, 16, 2, 64, device='cpu')
    k, table, lengths = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16), torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match='neither'):
        ha.paged_append(c, k, k, table, lengths, return_keys=Neither())
    with pytest.raises(RuntimeError):                        # (two elements: torch says which)
        ha.paged_append(c, k, k, table, lengths, return_keys=torch.zeros(2))
