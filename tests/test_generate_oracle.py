"""Generation against the whole model in 64 bits, written out plainly, with scores whose spread makes attention look at where keys lie and which they are.

The decoder's own weights, N(0, 0.02), give scores of 0.1 and attention that is nearly a mean, whatever the positions.  Here the rows of queries and keys are taken
five times: scores have a standard deviation of 2.5 in every block.

Tolerance.  fp16 activations: a rounding is off by 2^-11 / sqrt(3) of the value in the mean.  Queries and keys take three each (norm, projection, rotation), so that a
score of 2.5 carries sqrt(6) * 2.8e-4 * 2.5 = 1.7e-3, and a block's output, with the roundings of its own, about 2.2e-3; four blocks, added up as independent and each
turning what it is given by as much as its scores are steep (about 2), 5e-3 of the logits' norm.  BOUND is twice that.  The mistakes that a cached step can make are planted in the oracle: the
least of them moves the logits seven times as far."""
import pytest
import torch

from hyperattention_b200.llm import ChatGLM2ShapedDecoder, DecoderCache, chatglm2_config

BOUND = 1e-2
HEADS, GROUPS, DIM = 4, 2, 128
F64 = torch.float64
MISTAKES = ['queries off by one', 'keys off by one', 'both off by one', 'no rotation', 'queries not rotated', 'newest key missing', 'first key missing',
            'mean of the values']


def model(device):
    cfg = chatglm2_config(num_layers=4, hidden_size=256, num_attention_heads=HEADS, kv_channels=DIM, multi_query_group_num=GROUPS, ffn_hidden_size=512,
                          padded_vocab_size=1000)
    m = ChatGLM2ShapedDecoder(cfg, seed=1, device='cpu', dtype=torch.float16).eval()
    with torch.no_grad():
        for layer in m.transformer.encoder.layers:
            layer.self_attention.query_key_value.weight[:(HEADS + GROUPS) * DIM].mul_(5)
    return m.to(device)


def oracle(m, ids, late, mistake=None):
    """Logits [n, vocab] of one sequence ids [n] in 64 bits on the CPU; the mistake befalls the positions from `late` on."""
    c, w = m.config, {k: v.cpu().double() for k, v in m.state_dict().items()}
    n, rot = ids.shape[0], DIM // 2
    pos = torch.arange(n, dtype=F64)
    after = pos >= late
    inv = (10000.0 * c.rope_ratio) ** -(torch.arange(0, rot, 2, dtype=F64) / rot)

    def turn(x, p):
        z = torch.view_as_complex(x[..., :rot].unflatten(-1, (-1, 2)).contiguous()) * torch.polar(torch.ones(n, rot // 2, dtype=F64), p[:, None] * inv)[:, None]
        return torch.cat([torch.view_as_real(z).flatten(-2), x[..., rot:]], -1)

    def norm(x, weight):
        return weight * x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + c.layernorm_epsilon)

    at = {None: (0, 0), 'queries off by one': (1, 0), 'keys off by one': (0, 1), 'both off by one': (1, 1)}.get(mistake, (0, 0))
    qp, kp = pos + at[0] * after, pos + at[1] * after
    if mistake == 'no rotation':
        kp = pos * ~after
    if mistake in ('no rotation', 'queries not rotated'):
        qp = pos * ~after
    sees = pos[None] <= pos[:, None]
    if mistake == 'newest key missing':
        sees &= ~(after[:, None] & (pos[None] == pos[:, None]))
    if mistake == 'first key missing':
        sees &= ~(after[:, None] & (pos[None] == 0))
    x = w['transformer.embedding.weight'][ids.cpu()]
    for i in range(c.num_layers):
        p = f'transformer.encoder.layers.{i}.'
        h = norm(x, w[p + 'input_layernorm.weight']) @ w[p + 'self_attention.query_key_value.weight'].T + w[p + 'self_attention.query_key_value.bias']
        q, k, v = [t.unflatten(-1, (-1, DIM)) for t in h.split([HEADS * DIM, GROUPS * DIM, GROUPS * DIM], -1)]
        q, k = turn(q, qp).unflatten(1, (GROUPS, -1)), turn(k, kp)
        s = (torch.einsum('qhgd,khd->hgqk', q, k) * DIM ** -0.5).masked_fill(~sees, -torch.inf)
        a = s.softmax(-1)
        if mistake == 'mean of the values':
            a = torch.where(after[:, None], sees / sees.sum(-1, keepdim=True), a)
        x = x + torch.einsum('hgqk,khd->qhgd', a, v).flatten(1) @ w[p + 'self_attention.dense.weight'].T
        u, g = (norm(x, w[p + 'post_attention_layernorm.weight']) @ w[p + 'mlp.dense_h_to_4h.weight'].T).chunk(2, -1)
        x = x + (torch.nn.functional.silu(u) * g) @ w[p + 'mlp.dense_4h_to_h.weight'].T
    return norm(x, w['transformer.encoder.final_layernorm.weight']) @ w['transformer.output_layer.weight'].T


def rel(a, b):
    return ((a.cpu().double() - b).norm() / b.norm()).item()


def tokens(*shape):
    return torch.randint(0, 1000, shape, generator=torch.Generator().manual_seed(3))


def shortfall(m, ids, prompt):
    """How far the logit of any token behind the prompt is from the largest of its place (0 for the most probable ones), in units of the logits' standard deviation."""
    z = oracle(m, ids, 0)[prompt - 1:-1]
    chosen = z.gather(1, ids[prompt:].cpu()[:, None])[:, 0]
    return ((z.amax(-1) - chosen) / z.std(-1)).max().item()


# The logits' errors are BOUND of their standard deviation: of a thousand, the largest lies within five of those, and two of them part a chosen one from the largest.
SHORT = 2 * 5 * BOUND


def test_the_oracle_is_the_model():
    m = model('cpu').float()
    ids = tokens(60)
    with torch.no_grad():
        assert rel(m(ids[None])[0], oracle(m, ids, 0)) < 1e-5                   # 32 bits, and its angles


@pytest.mark.parametrize('mistake', MISTAKES)
def test_mistakes_show(mistake):
    """what the tests below would not let pass: by the logits of five cached positions, and by the tokens that are picked"""
    m = model('cpu')
    ids = tokens(60)
    right = oracle(m, ids, 0)[55:]
    assert rel(oracle(m, ids, 55, mistake)[55:], right) > 5 * BOUND
    worst = 0.0
    for prompt in (37, 5, 20):
        ids = tokens(40)[:prompt]
        for _ in range(8):
            ids = torch.cat([ids, oracle(m, ids, prompt, mistake)[-1:].argmax(-1)])
        worst = max(worst, shortfall(m, ids, prompt))
    assert worst > 3 * SHORT
    if mistake == MISTAKES[0]:
        ids = tokens(40)[:20]
        for _ in range(8):
            ids = torch.cat([ids, oracle(m, ids, 20)[-1:].argmax(-1)])
        assert shortfall(m, ids, 20) == 0


@pytest.mark.gpu
@pytest.mark.parametrize('page', [16, 20])
@pytest.mark.parametrize('parts', [(55, 1, 3, 1), (7, 48, 5), (1,) * 12 + (48,)])
def test_cached_positions(page, parts):
    """a prompt, then what follows over the pages: each part by itself"""
    m = model('cuda')
    ids = tokens(2, 60).cuda()
    cache = DecoderCache(m.config, 2, 60, page_size=page, dtype=torch.float16)
    want = torch.stack([oracle(m, s, 0) for s in ids])
    at = 0
    with torch.no_grad():
        for n in parts:
            got = m(ids[:, at:at + n], cache)
            assert rel(got, want[:, at:at + n]) < BOUND, (at, n)
            at += n
    assert cache.held.tolist() == [60, 60]


@pytest.mark.gpu
@pytest.mark.parametrize('graph', [True, False])
@pytest.mark.parametrize('counts', [None, (37, 5, 20)])
def test_generated_tokens(graph, counts):
    """every token is the most probable one behind its own sequence, with and without padded prompts"""
    m = model('cuda')
    ids = tokens(3, 37).cuda()
    cnt = None if counts is None else torch.tensor(counts, dtype=torch.int32, device='cuda')
    out = m.generate(ids, 10, counts=cnt, graph=graph)
    assert out.shape == (3, 10)
    for b, c in enumerate(counts or (37,) * 3):
        assert shortfall(m, torch.cat([ids[b, :c], out[b]]), c) <= SHORT


@pytest.mark.gpu
def test_padded_continuation():
    """a padded prompt, then padded tokens behind it: each sequence goes on from where it is"""
    m = model('cuda')
    ids = tokens(3, 60).cuda()
    cache = DecoderCache(m.config, 3, 64, page_size=16, dtype=torch.float16)
    held = [0, 0, 0]
    rows = [[], [], []]
    with torch.no_grad():
        for n, counts in ((30, (30, 4, 17)), (5, (1, 5, 3)), (1, None), (8, (8, 1, 5))):
            step = torch.zeros(3, n, dtype=torch.int64, device='cuda')
            for b, c in enumerate(counts or (n,) * 3):
                step[b, :c] = ids[b, held[b]:held[b] + c]
            got = m(step, cache, None if counts is None else torch.tensor(counts, dtype=torch.int32, device='cuda'))
            for b, c in enumerate(counts or (n,) * 3):
                rows[b].append(got[b, :c])
                held[b] += c
            assert cache.held.tolist() == held
    for b in range(3):
        want, at = oracle(m, ids[b, :held[b]], 0), 0
        for part in rows[b]:
            assert rel(part, want[at:at + len(part)]) < BOUND, (b, at)
            at += len(part)
