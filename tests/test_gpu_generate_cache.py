"""Generation into a caller's cache: room that is just enough, tables that name no page, counts out of range."""
import pytest
import torch

import hyperattention_b200 as ha
import test_generate_oracle as plain
from hyperattention_b200.llm import DecoderCache

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def model():
    return plain.model('cuda')


def _cache(m, batch, max_len):
    return DecoderCache(m.config, batch, max_len, page_size=16, dtype=torch.float16)


@pytest.mark.parametrize('graph', [True, False])
def test_room_for_all_but_the_last_token(model, graph):
    ids = plain.tokens(2, 37).cuda()
    want = model.generate(ids, 13, graph=False)
    cache = _cache(model, 2, 48)
    for new in (13, 20):
        with pytest.raises(AssertionError, match='the cache holds 48 tokens'):
            model.generate(ids, new, cache=cache, graph=graph)
    assert cache.length == 0 and not cache.held.any()
    assert torch.equal(model.generate(ids, 12, cache=cache, graph=graph), want[:, :12])
    assert cache.length == 48 and cache.held.tolist() == [48, 48]


@pytest.mark.parametrize('graph', [True, False])
@pytest.mark.parametrize('new', [3, 12])
def test_a_table_that_names_no_page(model, graph, new):
    """the steps that reach it, replayed or not, do not return tokens; the model is healthy again behind that"""
    ids = plain.tokens(1, 46).cuda()
    cache = _cache(model, 1, 64)
    cache.table[0, 2 if new == 3 else 3] = 99
    with pytest.raises(RuntimeError, match='outside'):
        model.generate(ids, new, cache=cache, graph=graph)
    torch.cuda.synchronize()
    try:
        ha.check_device_status()
    except RuntimeError:
        assert not graph                                     # (launches under way when a step's own call raised may report it once more)
    cache.clear()
    cache.table[0] = torch.tensor([3, 1, 0, 2], dtype=torch.int32)
    assert torch.equal(model.generate(ids, new, cache=cache, graph=graph), model.generate(ids, new, graph=False))


def test_counts_out_of_range(model):
    """as the operators take them: none below 0, all of the call's rows above; what the cache is said to hold is what was written"""
    ids = plain.tokens(2, 12).cuda()
    cache = _cache(model, 2, 64)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device='cuda')
    with torch.no_grad():
        model(ids[:, :5], cache, i32(5, 5))
        model(ids[:, 5:9], cache, i32(7, -3))
        assert cache.held.tolist() == [9, 5]
        got = model(torch.stack([ids[0, 9:12], ids[1, 5:8]]), cache)
    assert plain.rel(got[0], plain.oracle(model, ids[0], 0)[9:]) < plain.BOUND and plain.rel(got[1], plain.oracle(model, ids[1, :8], 0)[5:]) < plain.BOUND
