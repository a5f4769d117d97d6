"""What the operators of the paged cache refuse or report on the GPU, beyond the tests of test_gpu_paged.py."""
import math

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


@pytest.mark.parametrize('bits', [16, 4])
@pytest.mark.parametrize('columns', [0, 3, 5000])
def test_a_pool_without_pages(bits, columns):
    """sequences that hold nothing have empty rows; a page that a sequence needs is reported (5000 columns: by the list of tiles)"""
    cache = ha.PagedCache.allocate(0, 16, 2, 64, bits=bits)
    x = torch.ones(2, 1, 2, 64, dtype=torch.bfloat16, device='cuda')
    table, none = torch.zeros(2, columns, dtype=torch.int32, device='cuda'), torch.zeros(2, dtype=torch.int32, device='cuda')
    o, lse = ha.paged_attn_func(x, cache, table, none)
    k, v = ha.paged_gather(cache, table, none, 5)
    assert not o.any() and (lse == -math.inf).all() and not k.any() and not v.any()
    ha.check_device_status()
    for call in (lambda: ha.paged_attn_func(x, cache, table, none + 1), lambda: ha.paged_gather(cache, table, none + 1, 5), lambda: ha.paged_append(cache, x, x, table, none)):
        call()
        with pytest.raises(RuntimeError, match='outside'):
            ha.check_device_status()


def test_a_rotation_without_positions():
    """refused, not taken for no rotation; without elements to rotate, or without tokens, there is nothing to look up"""
    cache = ha.PagedCache.allocate(2, 16, 2, 64)
    x = torch.ones(1, 1, 2, 64, dtype=torch.bfloat16, device='cuda')
    table, length = torch.zeros(1, 2, dtype=torch.int32, device='cuda'), torch.zeros(1, dtype=torch.int32, device='cuda')
    rope = torch.empty(8, 32, 2, device='cuda')
    with pytest.raises(AssertionError, match='rope'):
        ha.paged_append(cache, x, x, table, length, rope=rope[:0], q=x)
    assert torch.equal(ha.paged_append(cache, x, x, table, length, rope=rope[:, :0].contiguous(), q=x), x)
    assert ha.paged_append(cache, x[:, :0], x[:, :0], table, length, rope=rope[:0], q=x[:, :0]).shape == (1, 0, 2, 64)
