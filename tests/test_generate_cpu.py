"""Generation without a GPU: what is refused before the prompt runs (past the checks, the cache's operators themselves refuse CPU tensors, by another message)."""
import pytest
import torch

from hyperattention_b200.llm import ChatGLM2ShapedDecoder, DecoderCache, chatglm2_config


@pytest.fixture(scope='module')
def model():
    cfg = chatglm2_config(num_layers=2, hidden_size=64, num_attention_heads=2, kv_channels=64, ffn_hidden_size=64, padded_vocab_size=50)
    return ChatGLM2ShapedDecoder(cfg, seed=1, dtype=torch.bfloat16).eval()


def _i32(*x):
    return torch.tensor(x, dtype=torch.int32)


@pytest.mark.parametrize('counts', [_i32(7, 0), _i32(-1, 7), _i32(8, 3), _i32(7), _i32(7, 3, 1), torch.tensor([7, 3]), _i32(7, 3)[:, None]],
                         ids=['none', 'negative', 'beyond the prompt', 'too few', 'too many', 'int64', 'two dimensions'])
@pytest.mark.parametrize('graph', [True, False])
def test_generate_refuses_counts(model, counts, graph):
    """a sequence without tokens has no last position; one behind the prompt's end would index logits that are not there"""
    with pytest.raises(AssertionError, match='counts'):
        model.generate(torch.zeros(2, 7, dtype=torch.int64), 3, counts=counts, graph=graph)


def test_generate_refuses_an_empty_prompt(model):
    with pytest.raises(AssertionError, match='prompt'):
        model.generate(torch.zeros(2, 0, dtype=torch.int64), 3)


@pytest.mark.parametrize('graph', [True, False])
@pytest.mark.parametrize('sq,new', [(7, 11), (12, 6), (17, 1), (1, 400)])
def test_generate_refuses_a_cache_that_is_too_small(model, graph, sq, new):
    """16 places: the prompt and all new tokens but the last must fit, whatever runs the steps; what does not fit is refused before anything is written"""
    cache = DecoderCache(model.config, 2, 16, page_size=8, device='cpu')
    with pytest.raises(AssertionError, match='the cache holds 16 tokens'):
        model.generate(torch.zeros(2, sq, dtype=torch.int64), new, cache=cache, graph=graph)
    assert cache.length == 0 and not cache.held.any()
    for sq, new in ((7, 10), (16, 1), (1, 16)):              # just enough: on to the operators
        with pytest.raises(AssertionError, match='CUDA'):
            model.generate(torch.zeros(2, sq, dtype=torch.int64), new, cache=cache, graph=graph)
        cache.clear()


def test_generate_refuses_the_cache_of_another_batch(model):
    cache = DecoderCache(model.config, 3, 16, page_size=8, device='cpu')
    with pytest.raises(AssertionError, match='another batch'):
        model.generate(torch.zeros(2, 20, dtype=torch.int64), 3, cache=cache)


def test_a_refused_call_adds_nothing(model):
    """the cache is as empty as before, and takes the prompt when the call is made as it should be"""
    cache = DecoderCache(model.config, 2, 16, page_size=8, device='cpu')
    for _ in range(3):
        with pytest.raises(AssertionError, match='no gradient|CUDA'):
            model(torch.zeros(2, 12, dtype=torch.int64), cache)
        assert cache.length == 0 and not cache.held.any()
