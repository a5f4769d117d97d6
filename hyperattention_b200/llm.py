"""ChatGLM2-style integration of HyperAttention: the attention-layer patch of the reference and a random-init decoder of
the ChatGLM2-6B shape to run it in (benchmark configuration 4).

* ``FastCoreAttention`` and ``patch_attention_layers`` mirror chatglm_fast_attention.py:8-70 and
  replace_llm_attention.py:6-44 of the reference: same constructor arguments, same layer-selection options, same
  [sq, b, heads, head_dim] calling convention, causal prefill only.
* ``ChatGLM2ShapedDecoder`` is written from the public description of the architecture (hidden 4096, 32 query heads of
  128, multi-query attention with 2 key/value groups, rotary embedding on half of each head, RMSNorm, SwiGLU MLP of
  13696, vocabulary 65024, 28 blocks), with the module nesting the patch expects
  (``model.transformer.encoder.layers[i].self_attention.core_attention``).  Weights are random (N(0, 0.02)); there
  is no checkpoint or tokenizer in this environment.  Everything outside the attention core is plain PyTorch.
* ``DecoderCache`` and ``ChatGLM2ShapedDecoder.generate`` go on from a prompt token by token: keys and values, rotated, in a paged cache
  of 16 or 4 bits (hyperattention_b200.paged), the new tokens' attention over its pages.
"""
import math
from types import SimpleNamespace

import torch
import torch.nn.functional as F

from .module import HyperAttention
from .ops import check_device_status
from .paged import PagedCache, paged_append, paged_attn_func

NUM_TOTAL_LAYERS = {
    'chatglm2-6b-32k': 28,
}


def select_patch_layers(num_total_layers, patch_config, num_patch_layers):
    """Indices of the blocks whose attention core is replaced (replace_llm_attention.py:10-35)."""
    n = num_total_layers if num_patch_layers < 0 else num_patch_layers
    t = num_total_layers
    table = {
        'last': lambda: range(t - 1, t - n - 1, -1),
        'first': lambda: range(n),
        'odd': lambda: range(1, t, 2),
        'even': lambda: range(0, t, 2),
        'odd_first': lambda: range(1, 2 * n, 2),
        'odd_last': lambda: range(t - 1, t - n, -1),
        'even_first': lambda: range(0, t, 2)[:n],
        'even_last': lambda: range(1, t, 2)[-n:],
    }
    if patch_config not in table:
        raise NotImplementedError(f"Invalid patch_config option: {patch_config}")
    return list(table[patch_config]())


class FastCoreAttention(torch.nn.Module):
    """Drop-in for the ChatGLM2 attention core backed by HyperAttention (chatglm_fast_attention.py:8-70)."""

    def __init__(self, config, layer_number, **kwargs):
        super().__init__()
        self.apply_query_key_layer_scaling = config.apply_query_key_layer_scaling
        self.attention_softmax_in_fp32 = config.attention_softmax_in_fp32 or self.apply_query_key_layer_scaling
        self.layer_number = max(1, layer_number)
        projection_size = config.kv_channels * config.num_attention_heads
        self.hidden_size_per_partition = projection_size
        self.hidden_size_per_attention_head = projection_size // config.num_attention_heads
        self.num_attention_heads_per_partition = config.num_attention_heads
        self.norm_factor = math.sqrt(self.hidden_size_per_attention_head)
        self.coeff = None
        if self.apply_query_key_layer_scaling:
            self.coeff = self.layer_number
            self.norm_factor *= self.coeff
        self.attention_dropout = torch.nn.Dropout(config.attention_dropout)
        # grouped_kv=True: the caller may hand over K/V with fewer heads than Q (multi-query / grouped-query models); K is then
        # hashed and sorted once per K/V head and never expanded.  False (default): heads already expanded, as the
        # reference's callers do (chatglm_fast_attention.py:53-58).
        self.grouped_kv = bool(kwargs.get('grouped_kv', False))
        self.attn_method = kwargs.get('attn_method')
        if self.attn_method != 'hyper':
            raise NotImplementedError("Invalid attn_method option")
        self.attn = HyperAttention(
            input_dim=self.hidden_size_per_attention_head,   # 128 for ChatGLM2 (hard-coded in the reference)
            lsh_num_projs=kwargs.get('lsh_num_projs'), block_size=kwargs.get('block_size'),
            sample_size=kwargs.get('sample_size'), min_seq_len=kwargs.get('min_seq_len'),
            smooth_block=kwargs.get('smooth_block'),
            **{k: v for k, v in kwargs.items() if k in ('grad_mode', 'merge_mode', 'rng', 'fused_causal')})

    def forward(self, query_layer, key_layer, value_layer, attention_mask):
        # [sq, b, heads, head_dim] -> [b, heads, sq, head_dim]
        query_layer, key_layer, value_layer = [t.permute(1, 2, 0, 3) for t in (query_layer, key_layer, value_layer)]
        assert attention_mask is None and query_layer.shape[2] == key_layer.shape[2], \
            'only causal prefill (no mask, equal query and key lengths) goes through HyperAttention'
        context_layer = self.attn(query_layer, key_layer, value_layer, causal=True)
        context_layer = context_layer.permute(2, 0, 1, 3)
        return context_layer.reshape(*context_layer.shape[:-2], self.hidden_size_per_partition)


def patch_attention_layers(model, model_name, patch_config, num_patch_layers, **kwargs):
    """Swaps ``core_attention`` of the selected blocks for FastCoreAttention (replace_llm_attention.py:6-44).
    ``num_total_layers`` may be passed to patch a model of the same structure with another depth."""
    total = kwargs.pop('num_total_layers', None) or NUM_TOTAL_LAYERS[model_name]
    indices = select_patch_layers(total, patch_config, num_patch_layers)
    if model_name != 'chatglm2-6b-32k':
        raise NotImplementedError(f'unsupported model {model_name}')
    print(f"patch_config: {patch_config}, attn_method: {kwargs['attn_method']}, num_patch_layers: {num_patch_layers}, "
          f"patch_indices: {indices}")
    ref = next(model.parameters())
    for i in indices:
        core = FastCoreAttention(model.config, i, **kwargs).to(device=ref.device, dtype=ref.dtype)
        model.transformer.encoder.layers[i].self_attention.core_attention = core
    return indices


# ------------------------------------------------------------------------------------------------
# a decoder of the ChatGLM2-6B shape
# ------------------------------------------------------------------------------------------------
def chatglm2_config(**over):
    cfg = dict(num_layers=28, hidden_size=4096, num_attention_heads=32, kv_channels=128, multi_query_group_num=2,
               ffn_hidden_size=13696, padded_vocab_size=65024, layernorm_epsilon=1e-5, rope_ratio=50.0,
               apply_query_key_layer_scaling=True, attention_softmax_in_fp32=True, attention_dropout=0.0)
    cfg.update(over)
    return SimpleNamespace(**cfg)


class RMSNorm(torch.nn.Module):
    def __init__(self, dim, eps):
        super().__init__()
        self.weight = torch.nn.Parameter(torch.ones(dim))
        self.eps = eps

    def forward(self, x):
        v = x.float().pow(2).mean(-1, keepdim=True)
        return (self.weight * (x.float() * torch.rsqrt(v + self.eps))).to(x.dtype)


class ExactCoreAttention(torch.nn.Module):
    """The stock attention core: exact causal softmax attention on [sq, b, heads, head_dim] tensors."""

    def __init__(self, config, layer_number):
        super().__init__()
        self.hidden = config.kv_channels * config.num_attention_heads

    def forward(self, q, k, v, attention_mask):
        q, k, v = [t.permute(1, 2, 0, 3) for t in (q, k, v)]
        o = F.scaled_dot_product_attention(q, k, v, is_causal=attention_mask is None and q.shape[2] == k.shape[2])
        o = o.permute(2, 0, 1, 3)
        return o.reshape(*o.shape[:-2], self.hidden)


def _rope_cache(seq_len, rot_dim, ratio, device, dtype):
    """cos/sin of the rotary angles for positions 0..seq_len-1 over rot_dim/2 frequency pairs."""
    base = 10000.0 * ratio
    inv = 1.0 / (base ** (torch.arange(0, rot_dim, 2, device=device, dtype=torch.float32) / rot_dim))
    ang = torch.outer(torch.arange(seq_len, device=device, dtype=torch.float32), inv)      # [sq, rot_dim/2]
    return torch.stack([ang.cos(), ang.sin()], dim=-1).to(dtype)                          # [sq, rot_dim/2, 2]


def _apply_rope(x, cache):
    """x [sq, b, heads, hn]; rotates consecutive element pairs of the first half of hn."""
    sq, b, h, hn = x.shape
    rot = cache.shape[1] * 2
    xr, xp = x[..., :rot], x[..., rot:]
    xr = xr.reshape(sq, b, h, rot // 2, 2)
    c = cache[:sq].view(sq, 1, 1, rot // 2, 2)
    out = torch.stack([xr[..., 0] * c[..., 0] - xr[..., 1] * c[..., 1], xr[..., 1] * c[..., 0] + xr[..., 0] * c[..., 1]], -1)
    return torch.cat([out.flatten(3), xp], dim=-1)


class DecoderCache:
    """Keys and values of every block for ``batch`` sequences of at most ``max_len`` tokens (rounded up to whole pages).

    ``held`` int32 [batch]: tokens of each sequence in the cache; ``length``: an upper bound of them that the host knows.  ``rope``: cosines and sines by
    position, fp32 (angles in 64 bits).  Sequence b has pages b * columns .. of the pool in order; any table of another kind will do as well."""

    def __init__(self, config, batch, max_len, page_size=64, bits=16, dtype=torch.bfloat16, device='cuda'):
        assert batch >= 1 and max_len >= 1 and page_size >= 1
        self.columns = -(-max_len // page_size)
        self.capacity = self.columns * page_size
        self.batch, self.length = batch, 0
        self.layers = [PagedCache.allocate(batch * self.columns, page_size, config.multi_query_group_num, config.kv_channels, dtype, bits, device)
                       for _ in range(config.num_layers)]
        self.table = torch.arange(batch * self.columns, dtype=torch.int32, device=device).view(batch, self.columns)
        self.held = torch.zeros(batch, dtype=torch.int32, device=device)
        rot = config.kv_channels // 2
        inv = (10000.0 * config.rope_ratio) ** -(torch.arange(0, rot, 2, device=device, dtype=torch.float64) / rot)
        ang = torch.outer(torch.arange(self.capacity, device=device, dtype=torch.float64), inv)
        self.rope = torch.stack([ang.cos(), ang.sin()], -1).float()

    def check(self, config, batch, more):
        """Refuses what the cache is not for: `batch` sequences of a model, `more` tokens behind those that it holds."""
        assert batch == self.batch and len(self.layers) == config.num_layers, 'the cache is for another batch or model'
        assert self.length + more <= self.capacity, f'the cache holds {self.capacity} tokens a sequence'

    def clear(self):
        self.length = 0
        self.held.zero_()


_CAPTURE_STREAMS = {}


class _Step:
    """What the blocks of one cached forward share."""

    def __init__(self, cache, n, counts, prompt):
        self.cache, self.counts, self.prompt = cache, counts, prompt
        # (counts as the operators take them: what is written is what the cache holds)
        self.total = cache.held + (n if counts is None else counts.clamp(0, n))


class SelfAttention(torch.nn.Module):
    def __init__(self, config, layer_number):
        super().__init__()
        self.heads, self.hn, self.groups = config.num_attention_heads, config.kv_channels, config.multi_query_group_num
        proj = self.heads * self.hn
        self.query_key_value = torch.nn.Linear(config.hidden_size, proj + 2 * self.groups * self.hn, bias=True)
        self.core_attention = ExactCoreAttention(config, layer_number)
        self.dense = torch.nn.Linear(proj, config.hidden_size, bias=False)

    def forward(self, x, rope, step=None, layer=0):
        sq, b, _ = x.shape
        qkv = self.query_key_value(x)
        q, k, v = qkv.split([self.heads * self.hn, self.groups * self.hn, self.groups * self.hn], dim=-1)
        q = q.view(sq, b, self.heads, self.hn)
        k = k.view(sq, b, self.groups, self.hn)
        v = v.view(sq, b, self.groups, self.hn)
        if step is None:
            q, k = _apply_rope(q, rope), _apply_rope(k, rope)
        else:
            cache, at = step.cache.layers[layer], step.cache
            q, k, v = [t.transpose(0, 1) for t in (q, k, v)]                     # [b, sq, heads, hn], as the cache's operators take them
            if not step.prompt:
                q = paged_append(cache, k, v, at.table, at.held, step.counts, at.rope, q)
                o, _ = paged_attn_func(q, cache, at.table, step.total, step.counts)
                return self.dense(o.transpose(0, 1).reshape(sq, b, -1))
            q, k = paged_append(cache, k, v, at.table, at.held, step.counts, at.rope, q, return_keys=True)
            q, k, v = [t.transpose(0, 1) for t in (q, k, v)]
        rep = self.heads // self.groups
        # multi-query: every key/value group serves heads/groups query heads; expanded before the core, as the
        # attention core of the original model expects equal head counts
        if not getattr(self.core_attention, 'grouped_kv', False):
            k = k.unsqueeze(3).expand(-1, -1, -1, rep, -1).reshape(sq, b, self.heads, self.hn)
            v = v.unsqueeze(3).expand(-1, -1, -1, rep, -1).reshape(sq, b, self.heads, self.hn)
        return self.dense(self.core_attention(q, k, v, None))


class MLP(torch.nn.Module):
    def __init__(self, config):
        super().__init__()
        self.dense_h_to_4h = torch.nn.Linear(config.hidden_size, 2 * config.ffn_hidden_size, bias=False)
        self.dense_4h_to_h = torch.nn.Linear(config.ffn_hidden_size, config.hidden_size, bias=False)

    def forward(self, x):
        a, g = self.dense_h_to_4h(x).chunk(2, dim=-1)
        return self.dense_4h_to_h(F.silu(a) * g)


class GLMBlock(torch.nn.Module):
    def __init__(self, config, layer_number):
        super().__init__()
        self.input_layernorm = RMSNorm(config.hidden_size, config.layernorm_epsilon)
        self.self_attention = SelfAttention(config, layer_number)
        self.post_attention_layernorm = RMSNorm(config.hidden_size, config.layernorm_epsilon)
        self.mlp = MLP(config)

    def forward(self, x, rope, step=None, layer=0):
        x = x + self.self_attention(self.input_layernorm(x), rope, step, layer)
        return x + self.mlp(self.post_attention_layernorm(x))


class _Encoder(torch.nn.Module):
    def __init__(self, config):
        super().__init__()
        self.layers = torch.nn.ModuleList([GLMBlock(config, i + 1) for i in range(config.num_layers)])
        self.final_layernorm = RMSNorm(config.hidden_size, config.layernorm_epsilon)


class _Transformer(torch.nn.Module):
    def __init__(self, config):
        super().__init__()
        self.embedding = torch.nn.Embedding(config.padded_vocab_size, config.hidden_size)
        self.encoder = _Encoder(config)
        self.output_layer = torch.nn.Linear(config.hidden_size, config.padded_vocab_size, bias=False)


class ChatGLM2ShapedDecoder(torch.nn.Module):
    """Random-init decoder of the ChatGLM2-6B shape; ``forward(input_ids [b, sq]) -> logits [b, sq, vocab]`` (prefill)."""

    def __init__(self, config=None, seed=0, last_token_logits_only=False, device=None, dtype=None):
        super().__init__()
        self.config = config or chatglm2_config()
        with torch.device(device or 'cpu'):
            self.transformer = _Transformer(self.config)
        if dtype is not None:
            self.to(dtype=dtype)
        self.last_only = last_token_logits_only
        dev = next(self.parameters()).device
        g = torch.Generator(device=dev).manual_seed(seed)
        with torch.no_grad():
            for name, prm in self.named_parameters():
                if prm.dim() >= 2:
                    prm.copy_(torch.randn(prm.shape, generator=g, device=dev, dtype=torch.float32) * 0.02)
                elif name.endswith('bias'):
                    prm.zero_()

    def forward(self, input_ids, cache=None, counts=None):
        """Logits of a prompt.  With a DecoderCache, the tokens go on from what it holds, and are in it afterwards: into an empty cache a prompt of any length
        (its attention is the blocks' own), behind that a few tokens a sequence (theirs goes over the pages).  counts: int32 [b], tokens of each
        sequence where input_ids are padded on the right; logits of the padding mean nothing."""
        b, sq = input_ids.shape
        if cache is None:
            return self._run(input_ids, None)
        cache.check(self.config, b, sq)
        logits = self._run(input_ids, _Step(cache, sq, counts, cache.length == 0))
        cache.length += sq                                       # (a call that was refused on the way has added nothing)
        return logits

    def _run(self, input_ids, step):
        sq = input_ids.shape[1]
        x = self.transformer.embedding(input_ids).transpose(0, 1).contiguous()      # [sq, b, hidden]
        rope = None if step is not None else _rope_cache(sq, self.config.kv_channels // 2, self.config.rope_ratio, x.device, x.dtype)
        for i, layer in enumerate(self.transformer.encoder.layers):
            x = layer(x, rope, step, i)
        if step is not None:
            step.cache.held.copy_(step.total)
        x = self.transformer.encoder.final_layernorm(x)
        if self.last_only and (step is None or step.counts is None):
            x = x[-1:]
        return self.transformer.output_layer(x).transpose(0, 1)

    @torch.no_grad()
    def generate(self, input_ids, new_tokens, counts=None, cache=None, page_size=64, bits=16, graph=True):
        """The most probable new_tokens tokens behind a prompt, one by one: int64 [b, new_tokens].  counts: int32 [b] prompt lengths, 1 .. sq, where input_ids are
        padded on the right (their values are read on the host).  cache: an empty DecoderCache to use, with room for the prompt and
        all new tokens but the last; made for the call otherwise.  graph: the steps behind the second token replay a CUDA graph.  The tokens are there when
        it returns; what a kernel reported (a table that names no page) is raised."""
        b, sq = input_ids.shape
        assert sq >= 1, 'a prompt has a token at least'
        if counts is not None:
            assert counts.shape == (b,) and counts.dtype == torch.int32, 'counts must be int32 [batch]'
            # (not under a capture, where nothing can be read: the index below stays within the prompt all the same)
            if not (counts.is_cuda and torch.cuda.is_current_stream_capturing()):
                assert all(1 <= c <= sq for c in counts.tolist()), 'counts must be between 1 and the length of the padded prompts'
        w = self.transformer.output_layer.weight
        if cache is None:
            cache = DecoderCache(self.config, b, sq + new_tokens, page_size, bits, w.dtype, w.device)
        assert cache.length == 0, 'the cache is not empty'
        cache.check(self.config, b, sq + max(new_tokens - 1, 0))                 # (replayed steps do not pass forward's own check)
        out = torch.empty(b, new_tokens, dtype=torch.int64, device=input_ids.device)
        if new_tokens == 0:
            return out
        with torch.cuda.device_of(w):                            # (whichever device is current: streams and captures are the model's)
            self._greedy(input_ids, counts, cache, out, graph)
            if not torch.cuda.is_current_stream_capturing():
                check_device_status(w.device)                    # (a replay does not look at the status words)
        return out

    def _greedy(self, input_ids, counts, cache, out, graph):
        b, new_tokens = out.shape
        sq = input_ids.shape[1]
        logits = self(input_ids, cache, counts)
        last = logits[:, -1] if counts is None else logits[torch.arange(b, device=logits.device), counts.long().clamp(1, sq) - 1]
        ids = last.argmax(-1, keepdim=True)
        out[:, :1] = ids
        replay = None
        for i in range(1, new_tokens):
            if replay is not None:
                cache.length += 1
                replay.replay()
            else:
                ids.copy_(self(ids, cache)[:, -1].argmax(-1, keepdim=True))
                if graph and i + 2 < new_tokens:
                    torch.cuda.current_stream().synchronize()
                    replay = torch.cuda.CUDAGraph()
                    # (the capture's own stream, one a device: torch's default belongs to the device of the process's first capture)
                    if ids.device not in _CAPTURE_STREAMS:
                        _CAPTURE_STREAMS[ids.device] = torch.cuda.Stream()
                    with torch.cuda.graph(replay, stream=_CAPTURE_STREAMS[ids.device]):
                        ids.copy_(self._run(ids, _Step(cache, 1, None, False))[:, -1].argmax(-1, keepdim=True))
            out[:, i:i + 1] = ids
