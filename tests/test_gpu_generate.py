"""Generation with the paged cache: the cached decoder against the one that runs the whole prompt, captured against eager steps, padded prompts, 4 bits."""
import pytest
import torch

from hyperattention_b200.llm import ChatGLM2ShapedDecoder, DecoderCache, chatglm2_config, patch_attention_layers


def _small(device, dtype, **over):
    cfg = chatglm2_config(**dict(dict(num_layers=4, hidden_size=256, num_attention_heads=4, kv_channels=128, ffn_hidden_size=512, padded_vocab_size=1000), **over))
    return ChatGLM2ShapedDecoder(cfg, seed=1, device=device, dtype=dtype).eval()


def _rel(a, b):
    return ((a.float() - b.float()).norm() / b.float().norm()).item()


def test_cached_decoder_refuses_without_cuda():
    m = _small('cpu', torch.bfloat16)
    with pytest.raises(AssertionError, match='CUDA'), torch.no_grad():
        m(torch.zeros(1, 3, dtype=torch.int64), DecoderCache(m.config, 1, 8, device='cpu'))


def test_uncached_decoder_is_as_before():
    m = _small('cpu', torch.float32)
    ids = torch.randint(0, 1000, (2, 20), generator=torch.Generator().manual_seed(0))
    with torch.no_grad():
        assert m(ids).shape == (2, 20, 1000)


@pytest.mark.gpu
@pytest.mark.parametrize('page', [16, 20])
@pytest.mark.parametrize('groups', [2, 4])
def test_cached_logits(page, groups):
    """prompt, then one token, three tokens and one: the logits of the whole sequence at once (bf16 activations: a few steps of 2^-8 through four blocks)"""
    m = _small('cuda', torch.bfloat16, multi_query_group_num=groups)
    ids = torch.randint(0, 1000, (2, 60), device='cuda', generator=torch.Generator(device='cuda').manual_seed(3))
    cache = DecoderCache(m.config, 2, 60, page_size=page)
    with torch.no_grad():
        want = m(ids)
        got, at = [], 0
        for n in (55, 1, 3, 1):
            got.append(m(ids[:, at:at + n], cache))
            at += n
        assert cache.held.tolist() == [60, 60] and cache.length == 60
        assert _rel(torch.cat(got, 1), want) < 2e-2
        with pytest.raises(AssertionError, match='holds'):
            m(ids[:, :30], cache)
        cache.clear()
        assert _rel(m(ids, cache), want) < 2e-2
    with pytest.raises(AssertionError):
        m.generate(ids, 2, cache=cache)


@pytest.mark.gpu
def test_generate_graph_and_padding():
    m = _small('cuda', torch.bfloat16)
    g = torch.Generator(device='cuda').manual_seed(5)
    ids = torch.randint(0, 1000, (3, 37), device='cuda', generator=g)
    eager = m.generate(ids, 12, graph=False)
    assert eager.shape == (3, 12) and torch.equal(m.generate(ids, 12), eager)
    cache = DecoderCache(m.config, 3, 64, page_size=16)
    for _ in range(2):                                      # the same cache again: a new graph, the old one's memory gone
        cache.clear()
        assert torch.equal(m.generate(ids, 12, cache=cache), eager)
    # the first token is the whole model's
    with torch.no_grad():
        assert torch.equal(m(ids)[:, -1].argmax(-1), eager[:, 0])
    # right padding: each sequence as if it were alone (the same products, in other batches: ties of bf16 logits apart)
    counts = torch.tensor([37, 5, 20], dtype=torch.int32, device='cuda')
    cache = DecoderCache(m.config, 3, 40, page_size=16)
    with torch.no_grad():
        logits = m(ids, cache, counts)
        assert cache.held.tolist() == [37, 5, 20]
        step = m(ids[:, :1], cache)
        for b, c in enumerate(counts.tolist()):
            alone = m(torch.cat([ids[b:b + 1, :c], ids[b:b + 1, :1]], 1))
            assert _rel(logits[b, c - 1], alone[0, c - 1]) < 2e-2 and _rel(step[b, 0], alone[0, c]) < 2e-2
    assert m.generate(ids, 1, counts=counts).shape == (3, 1) and m.generate(ids, 0).shape == (3, 0)


@pytest.mark.gpu
def test_generate_four_bits():
    """runs, repeats itself, and a step's logits stay near those of the 16-bit cache"""
    m = _small('cuda', torch.bfloat16)
    ids = torch.randint(0, 1000, (2, 50), device='cuda', generator=torch.Generator(device='cuda').manual_seed(6))
    a = m.generate(ids, 8, bits=4)
    assert torch.equal(a, m.generate(ids, 8, bits=4, graph=False))
    steps = []
    with torch.no_grad():
        for bits in (16, 4):
            cache = DecoderCache(m.config, 2, 64, bits=bits)
            m(ids, cache)
            steps.append(m(ids[:, :1], cache))
    assert torch.isfinite(steps[1]).all() and _rel(steps[1], steps[0]) < 0.2


@pytest.mark.gpu
def test_generate_behind_a_patched_prompt():
    """the prompt's attention by HyperAttention (exact at this length), un-expanded K/V heads, the steps over the pages"""
    m = _small('cuda', torch.bfloat16)
    ids = torch.randint(0, 1000, (1, 600), device='cuda', generator=torch.Generator(device='cuda').manual_seed(7))
    plain = m.generate(ids, 1)
    patch_attention_layers(m, 'chatglm2-6b-32k', 'last', 2, num_total_layers=4, attn_method='hyper', lsh_num_projs=8, block_size=256, sample_size=256,
                           min_seq_len=2048, smooth_block=False)
    for layer in m.transformer.encoder.layers:
        if hasattr(layer.self_attention.core_attention, 'grouped_kv'):
            layer.self_attention.core_attention.grouped_kv = True
    with torch.no_grad():
        want = m(torch.cat([ids, plain], 1))[:, -1]
        cache = DecoderCache(m.config, 1, 700)
        m(ids, cache)
        assert _rel(m(plain, cache)[:, -1], want) < 2e-2
    assert m.generate(ids, 5).shape == (1, 5)
