"""The calls of generation with a paged key/value cache, as cases that can be timed and compared.

A case is a dict of plain values:

  op        'append'  new keys and values are rotated and written to their pages, the queries rotated on the way (a 4-bit cache is read back as
                      dense rows, the values that it stands for)
            'attend'  attention of the last tokens over the cache: output and log-sum-exp
            'step'    both, one after the other: what one decoder block does for a token
  bits      16 or 4: how the cache is held
  batch, tokens       sequences, and new tokens of each
  context   tokens that the longest sequence holds before the new ones; spread 'ragged': the others hold between a sixteenth of it and all of it,
            'even': all of them
  heads, kv_heads, dim, dtype
  rot       elements at the start of each row that are rotated, in pairs
  page      tokens of a page

A cache is k, v [pages, kv_heads, page, dim], or for 4 bits codes uint8 [pages, kv_heads, page, dim / 2] and scales fp16
[pages, kv_heads, page, dim / 64, 2]; table int32 [batch, columns] names the pages of each sequence in order.
"""
import math

import torch

own = False

DTYPES = {'bf16': torch.bfloat16, 'fp16': torch.float16}
BASE = dict(op='attend', bits=16, batch=1, tokens=1, context=514, spread='even', heads=32, kv_heads=2, dim=128, rot=64, dtype='bf16', page=64)
MOST = 32 * 131072 * 64                    # elements of K that a drawn call takes at most: as many as layer_131k


def _case(**over):
    return dict(BASE, **over)


def listed():
    return [
        # one token of a short chat: one block's attention over the prompt, latency of one call
        _case(name='chat_515'),
        # a server's batch of chats of unequal lengths
        _case(name='batch_8k', batch=32, context=8191, spread='ragged'),
        # a layer with as many K/V heads as query heads at the benchmark's length
        _case(name='layer_131k', context=131071, kv_heads=32, dim=64, page=256),
        # four drafted tokens a sequence are looked at in one call
        _case(name='draft_12k_fp16', batch=8, tokens=4, context=12283, spread='ragged', heads=16, kv_heads=4, page=16, dtype='fp16'),
        # the short chat with the cache in 4 bits
        _case(name='chat_2051_int4', bits=4, context=2050),
        # long contexts in a batch: what a 4-bit cache is for
        _case(name='batch_32k_int4', bits=4, batch=64, context=32767, spread='ragged'),
        # the largest case: one layer, long context, 4 bits, half precision
        _case(name='layer_262k_int4_fp16', bits=4, context=262143, kv_heads=32, dim=64, rot=32, page=128, dtype='fp16'),
        # a batch's new tokens go to the cache of one block
        _case(name='append_32', op='append', batch=32, context=700, spread='ragged'),
        # a prompt of the prefill benchmark's length goes to the cache
        _case(name='append_prompt_32k', op='append', tokens=32768, context=0),
        # new tokens of a batch of short chats, 4 bits, read back
        _case(name='append_24_int4', op='append', bits=4, batch=24, context=75, spread='ragged', page=16),
        # two prompts of odd length, as many K/V heads as query heads, 4 bits, read back for the prompt's attention
        _case(name='append_prompt_8k_int4_fp16', op='append', bits=4, batch=2, tokens=8191, context=131, kv_heads=32, dim=64, rot=32, page=48, dtype='fp16'),
        # one token through a block: append, then attend
        _case(name='step_16_4k', op='step', batch=16, context=4095, spread='ragged'),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['attend', 'attend', 'attend', 'append', 'step'])
    bits = 16 if op == 'step' else rng.choice([16, 4])
    dim = rng.choice([64, 128, 128])
    kv_heads = rng.choice([1, 2, 2, 4, 8, 32])
    group = rng.choice([g for g in (1, 2, 4, 6, 8, 16, 32) if g * kv_heads <= 64])
    batch = _log_int(rng, 1, 64)
    c = dict(op=op, bits=bits, batch=batch, heads=kv_heads * group, kv_heads=kv_heads, dim=dim, rot=rng.choice([dim // 2, dim]),
             dtype=rng.choice(['bf16', 'bf16', 'fp16']), page=rng.choice([16, 32, 48, 64, 100, 128, 256]), spread=rng.choice(['even', 'ragged']))
    most = MOST // (batch * kv_heads * dim)                    # rows a sequence
    if op == 'append':
        prompt = rng.random() < 0.5
        c['tokens'] = _log_int(rng, 16, max(17, min(16384, most // 16))) if prompt else rng.choice([1, 1, 2, 5])
        c['context'] = rng.choice([0, _log_int(rng, 1, 1000)])
    else:
        c['tokens'] = rng.choice([1, 1, 1, 1, 2, 3, 5, 8])
        most = min(most, 10 * most // (group * c['tokens']))       # ... and no more products than batch_32k_int4
        c['context'] = _log_int(rng, 1, max(1, min(262143, most)))
    return _case(**c)


def _contexts(case):
    """Tokens that each sequence holds before the call: a fixed pattern, the first sequence the longest."""
    B, n = case['batch'], case['context']
    if case['spread'] == 'even':
        return [n] * B
    return [int(n * 16 ** -((b * 0.6180339887) % 1)) for b in range(B)]


# ---------------------------------------------------------------------------------------------------------------------
# the 4-bit form: groups of 64 elements; a 32-bit word holds 8 neighbours; where a row has two groups, their words alternate

def _quantise(x):
    """x fp32 [..., d] -> codes uint8 [..., d / 2], scales fp16 [..., d / 64, 2]."""
    g = x.unflatten(-1, (-1, 64))
    lo, hi = g.amin(-1), g.amax(-1)
    s, m = ((hi - lo) / torch.full_like(hi, 15)).half(), lo.half()        # (a division: by a number, torch multiplies by its reciprocal)
    sf, mf = s.float().unsqueeze(-1), m.float().unsqueeze(-1)
    q = torch.where(sf > 0, torch.round((g - mf) / sf).clamp(0, 15), torch.zeros_like(g)).to(torch.uint8)     # [..., groups, 64]
    q = q.unflatten(-1, (8, 8)).transpose(-3, -2).flatten(-3)                                                 # words of the groups in turn
    return q[..., 0::2] | (q[..., 1::2] << 4), torch.stack([s, m], -1)


def _values(codes, scales):
    """What codes and scales stand for, fp32 [..., d]."""
    q = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    q = q.unflatten(-1, (8, -1, 8)).transpose(-3, -2).flatten(-2).float()                                     # [..., groups, 64]
    return (q * scales[..., :1].float() + scales[..., 1:].float()).flatten(-2)


# ---------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    c = case
    g = torch.Generator(device='cuda').manual_seed(seed)
    B, n, H, Hk, d, ps, dt = c['batch'], c['tokens'], c['heads'], c['kv_heads'], c['dim'], c['page'], DTYPES[c['dtype']]
    held = _contexts(c)
    total = [h + n for h in held]
    need = [-(-t // ps) for t in total]
    pages = sum(need) + 3
    # pages in no order, as a server's pool hands them out; entries behind a sequence's last page name none
    order = torch.randperm(pages, generator=g, device='cuda').int()
    col = torch.arange(max(need), device='cuda')[None]
    first = torch.tensor([sum(need[:b]) for b in range(B)], device='cuda')[:, None]
    count = torch.tensor(need, device='cuda')[:, None]
    table = torch.where(col < count, order[(first + col).clamp(max=pages - 1)], torch.full_like(order[:1], -1)).contiguous()

    def normal(*shape):
        return torch.randn(*shape, generator=g, device='cuda')

    s = dict(case=c, table=table, held=torch.tensor(held, dtype=torch.int32, device='cuda'), total=torch.tensor(total, dtype=torch.int32, device='cuda'),
             rows=max(total))
    for name in ('k', 'v'):
        x = normal(pages, Hk, ps, d)
        if c['bits'] == 4:
            s[name + '_pages'], s[name + '_scales'] = _quantise(x)
        else:
            s[name + '_pages'], s[name + '_scales'] = x.to(dt), None
        del x
    # the projection's output: queries, keys and values of a token side by side
    qkv = normal(B, n, (H + 2 * Hk) * d)
    qkv[..., :H * d] *= 2
    s['q'], s['k'], s['v'] = [t.unflatten(-1, (-1, d)) for t in qkv.to(dt).split([H * d, Hk * d, Hk * d], -1)]
    # cosines and sines by position, angles in 64 bits
    inv = 500000.0 ** -(torch.arange(0, c['rot'], 2, device='cuda', dtype=torch.float64) / c['rot'])
    ang = torch.arange(max(total), device='cuda', dtype=torch.float64)[:, None] * inv
    s['rope'] = torch.stack([ang.cos(), ang.sin()], -1).float()
    if own:
        # the handle that a program keeps beside its pages: the same tensors, checked once
        import hyperattention_b200 as ha
        s['cache'] = ha.PagedCache(s['k_pages'], s['v_pages'], s['k_scales'], s['v_scales'], dtype=dt)
    return s


# ---------------------------------------------------------------------------------------------------------------------
def _rotate(x, rope):
    """x [B, n, h, d], rope [B, n, rot / 2, 2] -> fp32."""
    x, rot = x.float(), 2 * rope.shape[2]
    x0, x1 = x[..., 0:rot:2], x[..., 1:rot:2]
    c, s = rope[..., 0].unsqueeze(2), rope[..., 1].unsqueeze(2)
    return torch.cat([torch.stack([x0 * c - x1 * s, x1 * c + x0 * s], -1).flatten(-2), x[..., rot:]], -1)


def _append(s):
    c = s['case']
    pos = (s['held'][:, None] + torch.arange(c['tokens'], device='cuda')).long()
    page, slot = s['table'].long().gather(1, pos // c['page']), pos % c['page']
    rope = s['rope'][pos]
    for name, x in (('k', _rotate(s['k'], rope)), ('v', s['v'].float())):
        if c['bits'] == 4:
            codes, scales = _quantise(x)
            s[name + '_pages'][page, :, slot] = codes
            s[name + '_scales'][page, :, slot] = scales
        else:
            s[name + '_pages'][page, :, slot] = x.to(s['v'].dtype)
    return _rotate(s['q'], rope).to(s['q'].dtype)


def _dense(s, name):
    """fp32 [B, kv_heads, rows, d] of the sequences' rows, zero behind each one's last."""
    at = s['table'].long().clamp(min=0)
    x = s[name + '_pages'][at]
    x = _values(x, s[name + '_scales'][at]) if s['case']['bits'] == 4 else x.float()
    x = x.transpose(1, 2).flatten(2, 3)[:, :, :s['rows']]
    return x.masked_fill((torch.arange(s['rows'], device='cuda') >= s['total'][:, None])[:, None, :, None], 0)


def _attend(s, q):
    c = s['case']
    n = c['tokens']
    k, v = _dense(s, 'k'), _dense(s, 'v')
    q = q.float().unflatten(2, (c['kv_heads'], -1)).permute(0, 2, 3, 1, 4).flatten(2, 3)          # [B, kv_heads, group * n, d]
    x = (q @ k.transpose(2, 3) * c['dim'] ** -0.5).unflatten(2, (-1, n))
    keys = s['total'][:, None] - n + 1 + torch.arange(n, device='cuda')                            # keys that token i sees
    x = x.masked_fill((torch.arange(s['rows'], device='cuda') >= keys[..., None])[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    p = (x - top).exp()
    l = p.sum(-1, keepdim=True)
    o = (p.flatten(2, 3) @ v).unflatten(2, (-1, n)) / l                                            # [B, kv_heads, group, n, d]
    return o.permute(0, 3, 1, 2, 4).flatten(2, 3).to(s['q'].dtype), (top + l.log()).squeeze(-1).flatten(1, 2)


def run(state):
    s, c = state, state['case']
    if own:
        import hyperattention_b200 as ha
        cache = s['cache']
        q = s['q'] if c['op'] == 'attend' else ha.paged_append(cache, s['k'], s['v'], s['table'], s['held'], rope=s['rope'], q=s['q'])
        if c['op'] == 'append':
            k, v = ha.paged_gather(cache, s['table'], s['total'], s['rows']) if c['bits'] == 4 else (s['k_pages'], s['v_pages'])
            return {'q': q, 'k': k, 'v': v}
        o, lse = ha.paged_attn_func(q, cache, s['table'], s['total'])
    else:
        q = s['q'] if c['op'] == 'attend' else _append(s)
        if c['op'] == 'append':
            k, v = [_dense(s, x).to(q.dtype) for x in 'kv'] if c['bits'] == 4 else (s['k_pages'], s['v_pages'])
            return {'q': q, 'k': k, 'v': v}
        o, lse = _attend(s, q)
    out = {'o': o, 'lse': lse}                                                                     # [B, n, heads, d], [B, heads, n]
    if c['op'] == 'step':
        out.update(q=q, k=s['k_pages'], v=s['v_pages'])
    return out


def work(case):
    c = case
    B, n, H, Hk, d = c['batch'], c['tokens'], c['heads'], c['kv_heads'], c['dim']
    held = _contexts(c)
    row = 2 * d if c['bits'] == 16 else d // 2 + d // 64 * 4                                       # bytes of a cached row
    nbytes = flops = 0
    if c['op'] != 'attend':
        nbytes += B * n * (2 * (2 * H + 2 * Hk) * d + 2 * Hk * row) + (max(held) + n - min(held)) * c['rot'] * 4
        flops += B * n * (H + Hk) * c['rot'] * 3
        if c['bits'] == 4:                                                                         # read back, dense
            nbytes += sum(h + n for h in held) * 2 * Hk * row + B * (max(held) + n) * 2 * Hk * d * 2
    if c['op'] != 'append':
        nbytes += sum(h + n for h in held) * 2 * Hk * row + B * n * H * (2 * 2 * d + 4)
        flops += 4 * H * d * sum(n * h + n * (n + 1) // 2 for h in held)
    return {'bytes': nbytes, 'flops': flops}


# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    """The same from the definitions in 64 bits, one sequence at a time."""
    c = case
    s = prepare(case, seed)
    B, n, H, Hk, d, ps = c['batch'], c['tokens'], c['heads'], c['kv_heads'], c['dim'], c['page']
    held, table, f64 = _contexts(c), s['table'].tolist(), torch.float64

    def turned(x, at):                                                     # x [n, h, d] at positions at ..: complex products
        rot = c['rot']
        w = torch.view_as_complex(s['rope'][at:at + n].to(f64))[:, None]
        z = torch.view_as_complex(x[..., :rot].to(f64).unflatten(-1, (-1, 2)).contiguous()) * w
        return torch.cat([torch.view_as_real(z).flatten(-2), x[..., rot:].to(f64)], -1)

    def held_as(x):                                                        # the 4-bit form's values of x [..., d], in 64 bits
        y = torch.empty_like(x)
        for a in range(0, d, 64):
            part = x[..., a:a + 64]
            lo, hi = part.min(-1, keepdim=True)[0], part.max(-1, keepdim=True)[0]
            step, base = ((hi - lo) / 15).half().to(f64), lo.half().to(f64)
            code = ((part - base) / step.clamp(min=1e-300)).round().clamp(0, 15)
            y[..., a:a + 64] = torch.where(step > 0, code * step + base, base)
        return y

    def read(name, b, rows):                                               # [Hk, rows, d] of the cache as it was prepared
        at = torch.tensor(table[b][:-(-rows // ps)] if rows else [], dtype=torch.long, device='cuda')
        x = s[name + '_pages'][at].transpose(0, 1).flatten(1, 2)[:, :rows]
        if c['bits'] == 16:
            return x.to(f64)
        sc = s[name + '_scales'][at].transpose(0, 1).flatten(1, 2)[:, :rows].to(f64)
        y = torch.empty(Hk, rows, d, dtype=f64, device='cuda')
        for e in range(d):                                                 # byte of element e: its word, words of two halves alternating
            word = (e % 64) // 8 * (d // 64) + e // 64
            y[..., e] = (x[..., word * 4 + e % 8 // 2] >> (4 * (e % 2)) & 15) * sc[..., e // 64, 0] + sc[..., e // 64, 1]
        return y

    out = {}
    if c['op'] != 'attend':
        out['q'] = torch.stack([turned(s['q'][b], held[b]) for b in range(B)])
        new = [{'k': turned(s['k'][b], held[b]), 'v': s['v'][b].to(f64)} for b in range(B)]
    if c['op'] == 'append' and c['bits'] == 4:
        for name in 'kv':
            out[name] = torch.zeros(B, Hk, s['rows'], d, dtype=f64, device='cuda')
            for b in range(B):
                out[name][b, :, :held[b]] = read(name, b, held[b])
                out[name][b, :, held[b]:held[b] + n] = held_as(new[b][name]).transpose(0, 1)
        return out
    if c['op'] != 'attend':
        for name in 'kv':
            out[name] = s[name + '_pages'].to(f64)
            for b in range(B):
                pos = torch.arange(held[b], held[b] + n)
                out[name][torch.tensor(table[b])[pos // ps].cuda(), :, (pos % ps).cuda()] = new[b][name]
        if c['op'] == 'append':
            return out
    if sum(held) * Hk * d > 1 << 29:
        return None
    o, lse = torch.empty(B, n, H, d, dtype=f64, device='cuda'), torch.empty(B, H, n, dtype=f64, device='cuda')
    for b in range(B):
        if c['op'] == 'step':                                              # what the cache holds of the new rows is rounded to its type
            at, q = held[b], out['q'][b].to(s['q'].dtype).to(f64)
            k, v = [torch.cat([read(x, b, at), new[b][x].to(s['q'].dtype).to(f64).transpose(0, 1)], 1) for x in 'kv']
        else:
            q, k, v = s['q'][b].to(f64), read('k', b, held[b] + n), read('v', b, held[b] + n)
        for i in range(n):
            keys = held[b] + 1 + i
            x = torch.einsum('hgd,hld->hgl', q[i].unflatten(0, (Hk, -1)), k[:, :keys]) / math.sqrt(d)
            z = torch.logsumexp(x, -1)
            o[b, i] = torch.einsum('hgl,hld->hgd', (x - z[..., None]).exp(), v[:, :keys]).flatten(0, 1)
            lse[b, :, i] = z.flatten()
    out.update(o=o, lse=lse)
    return out
