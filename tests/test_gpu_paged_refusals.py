"""What the operators of the paged cache refuse on the GPU, beyond the refusals of test_gpu_paged.py; nothing is launched."""
import pytest
import torch

import hyperattention_b200 as ha

pytestmark = pytest.mark.gpu


def test_scale_of_zero_is_refused():
    cache = ha.PagedCache.allocate(2, 16, 2, 64)
    cache.k.zero_(), cache.v.zero_()
    q = torch.ones(1, 1, 2, 64, dtype=torch.bfloat16, device='cuda')
    table, length = torch.zeros(1, 2, dtype=torch.int32, device='cuda'), torch.ones(1, dtype=torch.int32, device='cuda')
    launches = ha.launch_count()
    for scale in (0.0, 0, -0.0):
        with pytest.raises(AssertionError):
            ha.paged_attn_func(q, cache, table, length, softmax_scale=scale)
    assert ha.launch_count() == launches
