"""The paged key/value cache on the GPU against plain implementations in 64 bits.

Tolerances.  Appended rows: products and sums in 32 bits, one rounding: half a step of the type, and 4 * 2^-24 of the magnitudes.  In 4 bits the codes are
those of the formula in 32 bits, bit for bit.  Attention: a score s carries an error of at most e = 2 (d + 8) 2^-24 max sum |q_i k_ij| scale (products
exact, sums in 32 bits, possibly truncated; the factor scale and log2 e), so every weight a relative 2 e + 2^-20 (the exponential's own error and the
two divisions); weights are handed to the second product with a relative error of 2^-17 (16 bits: two terms of 8 or 11 bits) or, against (code - 7.5),
2^-11 (4 bits: one term of 11 bits); sums over L keys run through at most L / 64 + 64 additions in a row.  The output is rounded once: half a step."""
import math

import pytest
import torch

import hyperattention_b200 as ha
from hyperattention_b200 import _lib as L

pytestmark = pytest.mark.gpu
F64 = torch.float64
BF, HF = torch.bfloat16, torch.float16


def quantise(x):
    """Codes 0..15 [..., d], steps and offsets [..., d / 64] of rows x (fp32): the format's formula."""
    g = x.float().unflatten(-1, (-1, 64))
    lo, hi = g.amin(-1), g.amax(-1)
    s, m = ((hi - lo) / torch.full_like(hi, 15)).half(), lo.half()        # (by a number, torch would multiply by its reciprocal)
    bad = ~(torch.isfinite(s) & torch.isfinite(m))
    s, m = s.masked_fill(bad, 0), m.masked_fill(bad, math.nan)
    sf, mf = s.float()[..., None], m.float()[..., None]
    q = torch.where(sf > 0, torch.round((g - mf) / sf).clamp(0, 15), torch.zeros_like(g)).nan_to_num(0)
    return q.flatten(-2), s, m


def dequantised(x):
    q, s, m = quantise(x)
    return (q.unflatten(-1, (-1, 64)).double() * s.double()[..., None] + m.double()[..., None]).flatten(-2)


def make_cache(rows_k, rows_v, page, bits, dtype, gen, spare=2, poison=True, layout='heads'):
    """Pages (in no order, the rest of them poisoned) that hold rows_k, rows_v: lists of [len, Hk, d] tensors.  Returns (cache, table, values k, values v):
    the values are what the cache stands for, in 64 bits."""
    Hk, d = rows_k[0].shape[1:]
    lens = [r.shape[0] for r in rows_k]
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=gen)
    cols = max(need) + 1
    table = torch.full((len(lens), cols), -7, dtype=torch.int32)
    table[:, 0::2] = 1 << 30                              # entries behind the last page name nothing
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n].int()
        at += n
    if bits == 16:
        shape = (pages, Hk, page, d) if layout == 'heads' else (pages, page, Hk, d)
        store = [torch.full(shape, math.nan if poison else 0.0, dtype=dtype, device='cuda') for _ in 'kv']
        if layout != 'heads':
            store = [t.transpose(1, 2) for t in store]
        cache = ha.PagedCache(*store)
    else:
        codes = [torch.full((pages, Hk, page, d // 2), 0xff, dtype=torch.uint8, device='cuda') for _ in 'kv']
        scales = [torch.full((pages, Hk, page, d // 64, 2), math.nan if poison else 0.0, dtype=HF, device='cuda') for _ in 'kv']
        cache = ha.PagedCache(*codes, *scales, dtype=dtype)
    vals = []
    for name, rows in (('k', rows_k), ('v', rows_v)):
        out = []
        for b, r in enumerate(rows):
            r = r.cuda()
            pos = torch.arange(lens[b])
            pg, sl = table[b][pos // page].long().cuda(), (pos % page).cuda()
            if bits == 16:
                getattr(cache, name)[pg, :, sl] = r.to(dtype)
                out.append(r.to(dtype).double())
            else:
                q, s, m = quantise(r)
                q = q.to(torch.uint8).unflatten(-1, (d // 64, 8, 8)).transpose(-3, -2).flatten(-3)
                getattr(cache, name)[pg, :, sl] = q[..., 0::2] | (q[..., 1::2] << 4)
                getattr(cache, name + '_scales')[pg, :, sl] = torch.stack([s, m], -1)
                out.append(dequantised(r))
        vals.append(out)
    return cache, table.cuda(), vals[0], vals[1]


def reference(q, ks, vs, lens, counts, scale):
    """o, lse, sum p |v|, error bound of a score -- row by row in 64 bits."""
    B, n, H, d = q.shape
    Hk = ks[0].shape[1]
    o, lse = torch.zeros(B, n, H, d, dtype=F64, device='cuda'), torch.full((B, H, n), -math.inf, dtype=F64, device='cuda')
    mag, err = torch.zeros_like(o), torch.zeros(B, n, H, dtype=F64, device='cuda')
    for b in range(B):
        for i in range(n):
            keys = lens[b] - counts[b] + i + 1
            if i >= counts[b] or keys <= 0:
                continue
            x = q[b, i].double().unflatten(0, (Hk, -1))
            k, v = ks[b][:keys], vs[b][:keys]
            s = torch.einsum('hgd,lhd->hgl', x, k) * scale
            z = torch.logsumexp(s, -1)
            p = (s - z[..., None]).exp()
            o[b, i], lse[b, :, i] = torch.einsum('hgl,lhd->hgd', p, v).flatten(0, 1), z.flatten()
            mag[b, i] = torch.einsum('hgl,lhd->hgd', p, v.abs()).flatten(0, 1)
            err[b, i] = torch.einsum('hgd,lhd->hgl', x.abs(), k.abs()).amax(-1).flatten() * scale
    return o, lse, mag, err


def check(o, lse, want, bits, dtype, d, longest, groups_mag=None):
    wo, wl, mag, err = want
    empty = wl == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    assert not o.transpose(1, 2)[empty].any()
    # 4 bits: 7.5 steps at most stand beside a value; |m|, 15 s are within three spans of the group's extremes
    e = 2 * (d + 8) * 2 ** -24 * err * (4 if bits == 4 else 1)
    chain = longest / 64 + 64
    rel = 2 * e + 2 ** -20 + (2 ** -17 if bits == 16 else 2 ** -11) + chain * 2 ** -23
    big = mag if groups_mag is None else torch.maximum(mag, groups_mag)
    tol = torch.finfo(dtype).eps / 2 * wo.abs() + rel[..., None] * big + 2.0 ** -24 * (dtype == HF)
    off = (o.double() - wo).abs()
    assert (off <= tol).all(), (off / tol).max().item()
    tl = e.transpose(1, 2) + 2 ** -22 * (wl.abs() + 32) + chain * 2 ** -23
    assert ((lse.double() - wl).abs()[~empty] <= tl[~empty]).all()


def attend_case(bits, dtype, d, H, Hk, page, lens, n=1, counts=None, scale=None, seed=0, layout='heads', qscale=2.0, order='plain'):
    g = torch.Generator().manual_seed(seed)
    rk, rv = [[torch.randn(l, Hk, d, generator=g) for l in lens] for _ in 'kv']
    cache, table, ks, vs = make_cache(rk, rv, page, bits, dtype, g, layout=layout)
    B = len(lens)
    q = (torch.randn(B, n, H, d, generator=g) * qscale).to(dtype).cuda()
    if order == 'view':                                    # the heads of a wider projection's output
        wide = torch.randn(B, n, H + 2 * Hk, d, generator=g).to(dtype).cuda()
        wide[:, :, :H] = q
        q = wide[:, :, :H]
    elif order == 'heads':
        q = q.transpose(1, 2).contiguous().transpose(1, 2)
    elif order == 'odd':                                   # rows off every 16-byte boundary
        wide = torch.zeros(B, n, H, d + 1, dtype=dtype, device='cuda')
        wide[..., 1:] = q
        q = wide[..., 1:]
    length = torch.tensor(lens, dtype=torch.int32).cuda()
    cnt = None if counts is None else torch.tensor(counts, dtype=torch.int32).cuda()
    o, lse = ha.paged_attn_func(q, cache, table, length, cnt, scale)
    assert o.shape == (B, n, H, d) and o.dtype == dtype and lse.shape == (B, H, n) and lse.dtype == torch.float32
    want = reference(q, ks, vs, lens, counts or [n] * B, scale or d ** -0.5)
    big = None
    if bits == 4:                                          # rounding meets 7.5 steps: as much as half a group's span
        span = max([((r.unflatten(-1, (-1, 64)).amax(-1) - r.unflatten(-1, (-1, 64)).amin(-1)).max().item() if r.numel() else 0.0) for r in rv] + [0.0])
        big = torch.full_like(want[2], span)
    check(o, lse, want, bits, dtype, d, max(lens), big)
    return o, lse


@pytest.mark.parametrize('bits', [16, 4])
@pytest.mark.parametrize('dtype', [BF, HF])
@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('H,Hk', [(1, 1), (4, 4), (6, 2), (16, 1), (34, 2), (40, 2)])
def test_attention_heads_and_types(bits, dtype, d, H, Hk):
    attend_case(bits, dtype, d, H, Hk, 16, [70, 1, 0, 333, 128])


@pytest.mark.parametrize('bits', [16, 4])
@pytest.mark.parametrize('page', [1, 7, 16, 64, 100, 1000])
def test_attention_page_sizes(bits, page):
    attend_case(bits, BF, 128, 8, 2, page, [257, 64, 5, 1, 700])


@pytest.mark.parametrize('bits', [16, 4])
@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('length', [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 191, 255, 513, 4097, 20011])
def test_attention_lengths(bits, d, length):
    attend_case(bits, BF, d, 4, 2, 32, [length])


@pytest.mark.parametrize('bits', [16, 4])
@pytest.mark.parametrize('n', [2, 3, 8])
def test_attention_several_tokens(bits, n):
    """rows see one key more each; a sequence shorter than its tokens leaves its first rows empty; padding rows"""
    attend_case(bits, BF, 128, 8, 2, 16, [100, n, 1, 65, 0], n=n)
    attend_case(bits, HF, 64, 3, 3, 16, [100, n, 1, 65, 0, 31], n=n, counts=[n, 1, 0, n - 1, n, n])


@pytest.mark.parametrize('bits', [16, 4])
@pytest.mark.parametrize('order', ['view', 'heads', 'odd'])
def test_attention_query_strides(bits, order):
    attend_case(bits, BF, 128, 8, 2, 16, [90, 200], n=2, order=order)


def test_attention_token_major_pages():
    attend_case(16, BF, 128, 8, 4, 16, [90, 200], layout='tokens')


@pytest.mark.parametrize('bits', [16, 4])
def test_attention_large_and_small_scores(bits):
    attend_case(bits, BF, 128, 8, 2, 16, [500, 900], qscale=30.0)
    attend_case(bits, HF, 64, 8, 2, 16, [500, 900], qscale=1e-3, scale=0.01)


@pytest.mark.parametrize('bits', [16, 4])
def test_attention_more_lines_than_a_launch(bits):
    attend_case(bits, BF, 64, 2, 1, 16, [(37 * i) % 90 for i in range(500)])


def test_attention_weights_over_a_sink():
    """One key takes most of the weight and has small values: the long tail of small weights decides the output (fp16 weights are held large)."""
    for bits in (16, 4):
        g = torch.Generator().manual_seed(3)
        n, d = 6000, 64
        rk, rv = [torch.randn(n, 1, d, generator=g) * 0.1], [torch.randn(n, 1, d, generator=g) + 1.0]
        rk[0][0], rv[0][0] = 2.0, 1e-3
        cache, table, ks, vs = make_cache(rk, rv, 16, bits, HF, g)
        q = torch.full((1, 1, 4, d), 0.9, dtype=HF, device='cuda')
        o, lse = ha.paged_attn_func(q, cache, table, torch.tensor([n], dtype=torch.int32, device='cuda'))
        want = reference(q, ks, vs, [n], [1], d ** -0.5)
        big = torch.full_like(want[2], float((want[2] + 0).max()) + 7.5 * 0.5) if bits == 4 else None
        check(o, lse, want, bits, HF, d, n, big)
        assert ((o.double() - want[0]).norm() / want[0].norm()).item() < 2 ** -10


@pytest.mark.parametrize('bits', [16, 4])
def test_attention_values_that_are_no_numbers(bits):
    """A NaN that a sequence sees makes its rows NaN, in the K/V head that holds it; other sequences do not see it; an earlier token of the same call does not."""
    g = torch.Generator().manual_seed(5)
    lens, d = [150, 150, 40], 128
    rk, rv = [[torch.randn(l, 2, d, generator=g) for l in lens] for _ in 'kv']
    rk[0][149, 0, 3] = math.nan                             # seen by the last of three tokens alone
    rv[1][20, 1, 70] = math.inf
    cache, table, ks, vs = make_cache(rk, rv, 16, bits, BF, g)
    q = torch.randn(3, 3, 4, d, generator=g).to(BF).cuda()
    o, lse = ha.paged_attn_func(q, cache, table, torch.tensor(lens, dtype=torch.int32, device='cuda'))
    want = reference(q, ks, vs, lens, [3, 3, 3], d ** -0.5)[0]
    assert torch.equal(torch.isfinite(o), torch.isfinite(want.to(BF)))
    assert o[0, 2, :2].isnan().all() and o[0, :2].isfinite().all() and o[0, 2, 2:].isfinite().all() and o[2].isfinite().all()
    assert lse[0, :2, 2].isnan().all() and lse[0, :, :2].isfinite().all()
    ok = torch.isfinite(want)
    assert (o.double() - want)[ok].abs().max() < 0.05


@pytest.mark.parametrize('bits', [16, 4])
@pytest.mark.parametrize('dtype', [BF, HF])
@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('H,Hk,n', [(1, 1, 16), (2, 2, 5), (6, 2, 4), (8, 1, 3), (16, 4, 9), (5, 1, 17)])
def test_attention_tokens_share_an_item(bits, dtype, d, H, Hk, n):
    """packs of neighbouring tokens: whole and broken ones, sequences shorter than a pack, padding inside one"""
    attend_case(bits, dtype, d, H, Hk, 16, [n, 1, 0, 200 + n, 64, 3], n=n)
    attend_case(bits, dtype, d, H, Hk, 16, [n, 1, 9, 200 + n, 64, 3000], n=n, counts=[n, 1, 2, n - 1, 0, n])


@pytest.mark.parametrize('bits', [16, 4])
@pytest.mark.parametrize('what', [math.nan, math.inf])
@pytest.mark.parametrize('d', [64, 128])
def test_attention_tokens_of_an_item_keep_apart(bits, what, d):
    """a value that is no number in the last keys reaches the tokens that see its key, and no others, where they share an item"""
    g = torch.Generator().manual_seed(15)
    n, H, Hk = 8, 2, 1
    for length in (8, 70, 129):
        for back in (1, 3, 7):
            rk, rv = [[torch.randn(length, Hk, d, generator=g)] for _ in 'kv']
            rv[0][length - back, 0, 5] = what
            cache, table, ks, vs = make_cache(rk, rv, 16, bits, BF, g)
            q = torch.randn(1, n, H, d, generator=g).to(BF).cuda()
            o, lse = ha.paged_attn_func(q, cache, table, torch.tensor([length], dtype=torch.int32, device='cuda'))
            want, wl = reference(q, ks, vs, [length], [n], d ** -0.5)[:2]
            assert torch.equal(torch.isfinite(o), torch.isfinite(want)) and o[0, :n - back].isfinite().all() and not o[0, n - back:, :, 5].isfinite().any()
            ok = torch.isfinite(want)
            assert (o.double() - want)[ok].abs().max() < 0.05 and (lse.double() - wl).abs().max() < 1e-4
            # ... and a key
            rk[0][length - back, 0, 5] = what
            cache, table, ks, vs = make_cache(rk, rv, 16, bits, BF, g)
            o, lse = ha.paged_attn_func(q, cache, table, torch.tensor([length], dtype=torch.int32, device='cuda'))
            assert lse[0, :, :n - back].isfinite().all() and o[0, :n - back].isfinite().all() and o[0, n - back:, :, 5].isnan().all()


@pytest.mark.parametrize('dtype', [BF, HF])
@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('n', [1, 4, 16])
def test_attention_infinite_values(dtype, d, n):
    """an infinity among the values that a row sees is the column's sum, of its own sign, whatever its weight's rounding: of the first key, of equal weights, ..."""
    g = torch.Generator().manual_seed(25)
    for length in (1, 17, 200, 3000):
        for even in (True, False):
            rk, rv = [[torch.randn(length, 1, d, generator=g)] for _ in 'kv']
            if even:
                rk[0].zero_()
            rv[0][0, 0, 3], rv[0][length // 2, 0, 4], rv[0][length - 1, 0, 5] = math.inf, -math.inf, math.inf
            rv[0][length // 3, 0, 6], rv[0][length // 4, 0, 6] = math.inf, -math.inf if length > 4 else math.inf
            cache, table, ks, vs = make_cache(rk, rv, 16, 16, dtype, g)
            q = torch.randn(1, n, 2, d, generator=g).to(dtype).cuda()
            o, lse = ha.paged_attn_func(q, cache, table, torch.tensor([length], dtype=torch.int32, device='cuda'))
            want, wl = reference(q, ks, vs, [length], [n], d ** -0.5)[:2]
            empty = (wl == -math.inf).transpose(1, 2)
            assert not o[empty].any() and torch.equal(lse == -math.inf, wl == -math.inf)
            seen, whole = o[~empty].double(), want[~empty]
            assert torch.equal(seen.isnan(), whole.isnan()) and torch.equal(seen.isinf(), whole.isinf())
            assert torch.equal(seen[whole.isinf()], whole[whole.isinf()])
            # |o| < 8, as all values are: half a step is 4 eps at most, and the rest (weights in 16 bits or more, sums in 32) far below
            ok = whole.isfinite()
            assert (seen - whole)[ok].abs().max() < 8 * torch.finfo(dtype).eps


def test_attention_no_numbers_in_a_whole_warp():
    """NaN scores through all the keys of a warp's part, beside finite ones"""
    g = torch.Generator().manual_seed(5)
    rk, rv = [[torch.randn(64, 1, 64, generator=g)] for _ in 'kv']
    rk[0][16:32] = math.nan
    cache, table, _, _ = make_cache(rk, rv, 16, 16, BF, g)
    o, lse = ha.paged_attn_func(torch.ones(1, 1, 1, 64, dtype=BF, device='cuda'), cache, table, torch.tensor([64], dtype=torch.int32, device='cuda'))
    assert o.isnan().all() and lse.isnan().all()


@pytest.mark.parametrize('bits', [16, 4])
def test_attention_repeats_and_streams(bits):
    """the same bits again, on another stream, beside another call, and from a graph whose lengths and table change between replays"""
    g = torch.Generator().manual_seed(9)
    lens, d = [700, 64, 3000], 128
    rk, rv = [[torch.randn(l, 2, d, generator=g) for l in lens] for _ in 'kv']
    cache, table, ks, vs = make_cache(rk, rv, 16, bits, BF, g)
    q = torch.randn(3, 1, 32, d, generator=g).to(BF).cuda()
    length = torch.tensor(lens, dtype=torch.int32, device='cuda')
    o, lse = ha.paged_attn_func(q, cache, table, length)
    for _ in range(3):
        o2, lse2 = ha.paged_attn_func(q, cache, table, length)
        assert torch.equal(o, o2) and torch.equal(lse, lse2)
    side = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(4):
        for s in side:
            with torch.cuda.stream(s):
                outs.append(ha.paged_attn_func(q, cache, table, length))
    torch.cuda.synchronize()
    assert all(torch.equal(a, o) and torch.equal(b, lse) for a, b in outs)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    got = []
    for gr in graphs:
        with torch.cuda.graph(gr):
            got.append(ha.paged_attn_func(q, cache, table, length))
    graphs[0].replay()
    graphs[1].replay()
    graphs[0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, o) and torch.equal(b, lse) for a, b in got)
    length.copy_(torch.tensor([1, 0, 2999], dtype=torch.int32))
    table[[0, 2]] = table[[0, 2]].clone()
    graphs[0].replay()
    want = reference(q, ks, vs, [1, 0, 2999], [1, 1, 1], d ** -0.5)
    span = torch.full_like(want[2], 8.0) if bits == 4 else None
    check(*got[0], want, bits, BF, d, 2999, span)


def test_attention_beyond_32_bits_of_elements():
    """pages whose rows begin past 2^31 elements (and 2^32 bytes) of the pool"""
    page, d = 64, 128
    pages = (2 ** 31 // (page * d)) + 40
    pool = torch.zeros(pages, 1, page, d, dtype=BF, device='cuda')
    cache = ha.PagedCache(pool, pool)
    g = torch.Generator().manual_seed(2)
    table = torch.tensor([[pages - 1, 3, pages - 30, pages - 7]], dtype=torch.int32, device='cuda')
    held = torch.zeros(1, dtype=torch.int32, device='cuda')
    rows = torch.randn(1, 200, 1, d, generator=g).to(BF).cuda()
    ha.paged_append(cache, rows, rows, table, held)
    for c, p in enumerate(table[0].tolist()):
        part = rows[0, c * page:(c + 1) * page, 0]
        assert torch.equal(pool[p, 0, :part.shape[0]], part)
    q = torch.randn(1, 1, 4, d, generator=g).to(BF).cuda()
    o, lse = ha.paged_attn_func(q, cache, table, held + 200)
    x = rows[0].double()
    check(o, lse, reference(q, [x], [x], [200], [1], d ** -0.5), 16, BF, d, 200)
    k, v = ha.paged_gather(cache, table, held + 200, 201)
    assert torch.equal(k[0, 0, :200], rows[0, :, 0]) and torch.equal(k, v) and not k[0, 0, 200:].any()


def test_four_bits_beyond_32_bits_of_a_page():
    """one page whose rows lie past 2^31 bytes of it: appended, attended to, in whole runs"""
    page, d = 2 ** 25 + 128, 128
    codes, scales = [torch.zeros(1, 1, page, d // 2, dtype=torch.uint8, device='cuda') for _ in 'kv'], [torch.zeros(1, 1, page, 2, 2, dtype=HF, device='cuda') for _ in 'kv']
    cache = ha.PagedCache(*codes, *scales)
    g = torch.Generator().manual_seed(2)
    held, new, lead = 2 ** 25 + 10, 100, 2 ** 25 + 10
    table, i32 = torch.zeros(1, 1, dtype=torch.int32, device='cuda'), lambda x: torch.tensor([x], dtype=torch.int32, device='cuda')
    q = torch.randn(1, 1, 16, d, generator=g).to(BF).cuda()
    # keys along the sum of the queries: scores that outweigh the millions of zeros
    k = (q.float().sum(2, keepdim=True).cpu() + 0.5 * torch.randn(1, new, 1, d, generator=g)).to(BF).cuda()
    v = torch.randn(1, new, 1, d, generator=g).to(BF).cuda()
    ha.paged_append(cache, k, v, table, i32(held))
    o, lse = ha.paged_attn_func(q, cache, table, i32(held + new), softmax_scale=0.25)
    kk, vv = dequantised(k[0]), dequantised(v[0])
    s = torch.einsum('hd,ld->hl', q[0, 0].double(), kk[:, 0]) * 0.25                       # [heads, new]; all other scores and values are 0
    z = torch.logaddexp(torch.logsumexp(s, -1), torch.full((16,), math.log(lead), dtype=F64, device='cuda'))
    p = (s - z[:, None]).exp()
    want = p @ vv[:, 0]
    assert s.max() > 20 and (p.sum(-1) > 0.5).any()
    e = 8 * (d + 8) * 2 ** -24 * torch.einsum('hd,ld->hl', q[0, 0].double().abs(), kk[:, 0].abs()).amax(-1) * 0.25
    # as in check(): the score's error, the weights' rounding beside 7.5 steps (of spans below 8), chains of 2^25 / (128 * 400) tiles of additions
    tol = 2 ** -9 * want.abs() + (2 * e + 2 ** -11 + 1200 * 2 ** -23)[:, None] * 8
    assert ((o[0, 0].double() - want).abs() <= tol).all()
    assert ((lse[0, :, 0].double() - z).abs() <= e + 2 ** -22 * (z.abs() + 32) + 1200 * 2 ** -23).all()


# ---------------------------------------------------------------------------------------------------------------------
def rope_table(positions, rot, dtype=torch.float32):
    ang = torch.arange(positions, dtype=F64)[:, None] * 10000.0 ** -(torch.arange(0, rot, 2, dtype=F64) / max(rot, 1))
    return torch.stack([ang.cos(), ang.sin()], -1).to(dtype).cuda()


def rotated32(x, rope):
    """The rotation in 32 bits, every product and sum rounded: x [n, h, d], rope [n, rot / 2, 2]."""
    rot, x = 2 * rope.shape[1], x.float()
    c, s = rope[:, None, :, 0].float(), rope[:, None, :, 1].float()
    a, b = x[..., 0:rot:2], x[..., 1:rot:2]
    return torch.cat([torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2), x[..., rot:]], -1)


def append_case(bits, dtype, d, H, Hk, page, held, n, counts=None, rot=None, rope_dtype=torch.float32, order='plain', with_q=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    B = len(held)
    rk, rv = [[torch.randn(h, Hk, d, generator=g) for h in held] for _ in 'kv']
    room = [torch.cat([r, torch.full((n, Hk, d), 7.0)]) for r in rk], [torch.cat([r, torch.full((n, Hk, d), 7.0)]) for r in rv]
    cache, table, _, _ = make_cache(*room, page, bits, dtype, g, poison=False)
    qkv = torch.randn(B, n, H + 2 * Hk, d + (order == 'odd'), generator=g).to(dtype).cuda()
    if order == 'odd':
        qkv = qkv[..., 1:]
    if order == 'tokens':                                    # [n, B, heads, d], as the decoder holds its activations
        qkv = qkv.transpose(0, 1).contiguous().transpose(0, 1)
    q, k, v = qkv.split([H, Hk, Hk], 2)
    rope = None if rot is None else rope_table(max(held) + n, rot, rope_dtype)
    at = torch.tensor(held, dtype=torch.int32, device='cuda')
    cnt = None if counts is None else torch.tensor(counts, dtype=torch.int32, device='cuda')
    before = [t.clone() for t in (cache.k, cache.v)] + ([cache.k_scales.clone(), cache.v_scales.clone()] if bits == 4 else [])
    got = ha.paged_append(cache, k, v, table, at, cnt, rope, q if with_q else None, return_keys=True)
    expect = [t.clone() for t in before]
    for b in range(B):
        m = n if counts is None else max(0, min(counts[b], n))
        pos = torch.arange(held[b], held[b] + m)
        pg, sl = table[b].cpu()[pos // page].long().cuda(), (pos % page).cuda()
        rr = rope[held[b]:held[b] + m] if rope is not None else torch.zeros(m, 0, 2, device='cuda')
        kr, qr = rotated32(k[b, :m], rr), rotated32(q[b, :m], rr)
        for j, x in enumerate((kr, v[b, :m].float())):
            if bits == 16:
                expect[j][pg, :, sl] = x.to(dtype)
            else:
                c, s, mm = quantise(x)
                c = c.to(torch.uint8).unflatten(-1, (d // 64, 8, 8)).transpose(-3, -2).flatten(-3)
                expect[j][pg, :, sl] = c[..., 0::2] | (c[..., 1::2] << 4)
                expect[2 + j][pg, :, sl] = torch.stack([s, mm], -1)
        assert torch.equal(got[1][b, :m], kr.to(dtype)) and not got[1][b, m:].any()
        if with_q:
            assert torch.equal(got[0][b, :m], qr.to(dtype)) and not got[0][b, m:].any()
            # ... and against the formula in 64 bits
            if rope is not None and m:
                z = torch.view_as_complex(q[b, :m, :, :rot].double().unflatten(-1, (-1, 2)).contiguous()) * torch.view_as_complex(rr.double())[:, None]
                w = torch.view_as_real(z).flatten(-2)
                tol = torch.finfo(dtype).eps / 2 * w.abs() + (4 * 2 ** -24) * q[b, :m].double().abs().amax() * 2 + 2 ** -24
                assert ((got[0][b, :m, :, :rot].double() - w).abs() <= tol).all()
    if not with_q:
        assert got[0] is None
    after = [cache.k, cache.v] + ([cache.k_scales, cache.v_scales] if bits == 4 else [])
    for a, e in zip(after, expect):
        assert torch.equal(a.view(torch.int16) if a.dtype == HF else a, e.view(torch.int16) if e.dtype == HF else e)   # the new slots, and nothing else
    return cache, table, at


@pytest.mark.parametrize('bits', [16, 4])
@pytest.mark.parametrize('dtype', [BF, HF])
@pytest.mark.parametrize('d,rot', [(64, 64), (64, 2), (64, None), (128, 64), (128, 20), (128, 128), (128, 0)])
def test_append_rotations(bits, dtype, d, rot):
    append_case(bits, dtype, d, 6, 2, 16, [0, 15, 16, 33], 3, rot=rot)


@pytest.mark.parametrize('bits', [16, 4])
@pytest.mark.parametrize('page', [1, 7, 16, 100])
def test_append_pages_and_padding(bits, page):
    append_case(bits, BF, 128, 4, 4, page, [5, 0, 98], 21, counts=[21, 3, 0], rot=64)
    append_case(bits, BF, 64, 4, 4, page, [5, 0, 98], 1, counts=[-3, 9, 1], rot=64)


@pytest.mark.parametrize('bits', [16, 4])
@pytest.mark.parametrize('order', ['tokens', 'odd'])
def test_append_strides(bits, order):
    append_case(bits, BF, 128, 5, 1, 16, [5, 40], 4, rot=64, order=order)
    append_case(bits, HF, 64, 40, 4, 16, [5, 40], 2, rot=32, order=order, rope_dtype=HF)


def test_append_without_queries_and_long():
    append_case(16, BF, 128, 2, 2, 64, [3], 3000, rot=64, with_q=False)
    append_case(4, BF, 64, 32, 2, 64, [3], 999, rot=64, rope_dtype=BF)


@pytest.mark.parametrize('bits', [16, 4])
@pytest.mark.parametrize('dtype', [BF, HF])
@pytest.mark.parametrize('d,H,Hk', [(128, 18, 2), (128, 3, 3), (64, 34, 17), (64, 6, 2)])
def test_append_many_tokens(bits, dtype, d, H, Hk):
    """more tokens than are under way at once: blocks of fewer threads; padding among them, rows off their boundaries, none to rotate"""
    append_case(bits, dtype, d, H, Hk, 48, [5, 0], 420, counts=[401, 17], rot=d // 2)
    append_case(bits, dtype, d, H, Hk, 16, [1], 760, rot=d, rope_dtype=dtype, order='odd')
    append_case(bits, dtype, d, H, Hk, 100, [0, 3, 9], 300, order='tokens', with_q=False)


def test_append_empty_calls():
    cache = ha.PagedCache.allocate(2, 16, 2, 64)
    z = lambda *s: torch.zeros(*s, dtype=BF, device='cuda')
    table, at = torch.zeros(1, 1, dtype=torch.int32, device='cuda'), torch.zeros(1, dtype=torch.int32, device='cuda')
    assert ha.paged_append(cache, z(1, 0, 2, 64), z(1, 0, 2, 64), table, at, q=z(1, 0, 4, 64)).shape == (1, 0, 4, 64)
    o, lse = ha.paged_attn_func(z(1, 0, 4, 64), cache, table, at)
    assert o.shape == (1, 0, 4, 64) and lse.shape == (1, 4, 0)
    o, lse = ha.paged_attn_func(z(1, 1, 4, 64), cache, table[:, :0], at)                # a table without columns: no sequence holds anything
    assert not o.any() and (lse == -math.inf).all()
    k, v = ha.paged_gather(cache, table, at, 0)
    assert k.shape == (1, 2, 0, 64)
    e = torch.zeros(0, 1, dtype=torch.int32, device='cuda')
    assert ha.paged_attn_func(z(0, 1, 4, 64), cache, e, at[:0])[0].shape == (0, 1, 4, 64)


@pytest.mark.parametrize('value', ['constant', 'tiny', 'nan', 'inf', 'wide', 'offset'])
def test_four_bit_groups(value):
    """groups without a span, below fp16's range, beyond it, with values that are no numbers: the formula's codes, and what attention makes of them"""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(1, 4, 1, 128, generator=g)
    part = x[0, 1, 0, :64]
    if value == 'constant':
        part[:] = 1.25
    elif value == 'tiny':
        part *= 1e-9
    elif value == 'nan':
        part[7] = math.nan
    elif value == 'inf':
        part[7] = -math.inf
    elif value == 'wide':
        part *= 1e7
    else:
        part += 1000.0
    x = x.to(BF).cuda()
    cache = ha.PagedCache.allocate(1, 16, 1, 128, bits=4)
    table, at = torch.zeros(1, 1, dtype=torch.int32, device='cuda'), torch.zeros(1, dtype=torch.int32, device='cuda')
    ha.paged_append(cache, x, x, table, at)
    want = dequantised(x[0])                                                            # [4, 1, 128]
    k, v = ha.paged_gather(cache, table, at + 4, 4)
    torch.testing.assert_close(k[0].transpose(0, 1), want.to(torch.float32).to(BF), rtol=0, atol=0, equal_nan=True)
    assert torch.equal(k.view(torch.int16), v.view(torch.int16))
    got = cache.values()[0][0, 0, :4].double()
    torch.testing.assert_close(got, want[:, 0].float().double(), rtol=0, atol=0, equal_nan=True)
    q = torch.randn(1, 1, 2, 128, generator=g).to(BF).cuda()
    o, lse = ha.paged_attn_func(q, cache, table, at + 4)
    if value in ('nan', 'inf', 'wide'):
        assert o.isnan().all() and lse.isnan().all()
    else:
        span = (want.amax() - want.amin()).item()
        ref = reference(q, [want], [want], [4], [1], 128 ** -0.5)
        check(o, lse, ref, 4, BF, 128, 4, torch.maximum(ref[2], torch.full_like(ref[2], span)))


@pytest.mark.parametrize('bits', [16, 4])
@pytest.mark.parametrize('dtype', [BF, HF])
@pytest.mark.parametrize('d', [64, 128])
def test_gather(bits, dtype, d):
    g = torch.Generator().manual_seed(4)
    lens = [0, 1, 70, 200, 129]
    rk, rv = [[torch.randn(l, 3, d, generator=g) for l in lens] for _ in 'kv']
    cache, table, ks, vs = make_cache(rk, rv, 16, bits, dtype, g)
    length = torch.tensor(lens, dtype=torch.int32, device='cuda')
    for rows in (1, 100, 200, 209):
        for got, want in zip(ha.paged_gather(cache, table, length, rows), (ks, vs)):
            assert got.shape == (5, 3, rows, d) and got.is_contiguous()
            for b, l in enumerate(lens):
                m = min(l, rows)
                assert torch.equal(got[b, :, :m], want[b][:m].transpose(0, 1).float().to(dtype)) and not got[b, :, m:].any()


def test_shared_pages():
    """two sequences with the same first pages, and a sequence twice in one call"""
    g = torch.Generator().manual_seed(6)
    rk, rv = [[torch.randn(l, 2, 64, generator=g) for l in (50, 60)] for _ in 'kv']
    cache, table, ks, vs = make_cache(rk, rv, 16, 16, BF, g)
    table[1, :2] = table[0, :2]
    for t in (ks, vs):
        t[1][:32] = t[0][:32]
    both = torch.cat([table, table[:1]])
    q = torch.randn(3, 1, 4, 64, generator=g).to(BF).cuda()
    lens = [50, 60, 50]
    o, lse = ha.paged_attn_func(q, cache, both, torch.tensor(lens, dtype=torch.int32, device='cuda'))
    check(o, lse, reference(q, ks + ks[:1], vs + vs[:1], lens, [1] * 3, 64 ** -0.5), 16, BF, 64, 60)


@pytest.mark.parametrize('bits', [16, 4])
def test_bad_pages_are_reported(bits):
    """a page or position that does not exist: nothing out of range is touched (the kernels look before they read), the next call raises"""
    cache = ha.PagedCache.allocate(2, 16, 1, 64, bits=bits)
    for t in (cache.k, cache.v, cache.k_scales, cache.v_scales):
        if t is not None:
            t.zero_()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device='cuda')
    x = torch.ones(1, 2, 1, 64, dtype=BF, device='cuda')
    good, at = i32([[0, 1]]), i32([0])
    rope = rope_table(3, 64)
    calls = [lambda: ha.paged_append(cache, x, x, i32([[2, 1]]), at), lambda: ha.paged_append(cache, x, x, i32([[-1, 1]]), at),
             lambda: ha.paged_append(cache, x, x, good, i32([31])), lambda: ha.paged_append(cache, x, x, good, i32([-1])),
             lambda: ha.paged_append(cache, x, x, good, i32([2 ** 31 - 1])), lambda: ha.paged_append(cache, x, x, good, i32([2]), rope=rope),
             lambda: ha.paged_attn_func(x, cache, i32([[0, 2]]), i32([20])), lambda: ha.paged_attn_func(x, cache, good, i32([33])),
             lambda: ha.paged_attn_func(x, cache, i32([[-5, 1]]), i32([3])), lambda: ha.paged_gather(cache, i32([[0, 9]]), i32([20]), 20),
             lambda: ha.paged_gather(cache, good, i32([2 ** 31 - 1]), 20)]
    for call in calls:
        call()
        with pytest.raises(RuntimeError, match='outside'):
            ha.check_device_status()
    calls[0]()
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match='outside'):
        ha.paged_attn_func(x, cache, good, i32([1]))
    o, _ = ha.paged_attn_func(x, cache, good, i32([0]))                                  # healthy again
    assert not o.any()
    ha.paged_attn_func(x, cache, i32([[0, 99]]), i32([16]))                              # an entry that no key needs
    ha.paged_append(cache, x, x, i32([[0, 99]]), i32([14]))
    ha.check_device_status()


def test_refusals():
    cache = ha.PagedCache.allocate(2, 16, 2, 64)
    x = torch.ones(1, 2, 2, 64, dtype=BF, device='cuda')
    t, at = torch.zeros(1, 2, dtype=torch.int32, device='cuda'), torch.zeros(1, dtype=torch.int32, device='cuda')
    rope = rope_table(8, 64)
    bad = [lambda: ha.paged_append(cache, x.half(), x, t, at), lambda: ha.paged_append(cache, x, x[:, :1], t, at), lambda: ha.paged_append(cache, x[..., :32], x, t, at),
           lambda: ha.paged_append(cache, x, x, t.long(), at), lambda: ha.paged_append(cache, x, x, t, at.long()), lambda: ha.paged_append(cache, x, x, t[0], at),
           lambda: ha.paged_append(cache, x, x, t.cpu(), at), lambda: ha.paged_append(cache, x, x, t, at, counts=at.float()),
           lambda: ha.paged_append(cache, x, x, t, at, rope=rope.half()), lambda: ha.paged_append(cache, x, x, t, at, rope=rope_table(8, 66)),
           lambda: ha.paged_append(cache, x, x, t, at, q=torch.ones(1, 2, 3, 64, dtype=BF, device='cuda')),
           lambda: ha.paged_append(cache, x.clone().requires_grad_(), x, t, at), lambda: ha.paged_attn_func(x.clone().requires_grad_(), cache, t, at),
           lambda: ha.paged_attn_func(x[:, :, :1], cache, t, at), lambda: ha.paged_attn_func(x.float(), cache, t, at), lambda: ha.paged_attn_func(x, cache, t, at[:0]),
           lambda: ha.paged_gather(cache, t, at, -1)]
    launches = ha.launch_count()
    for call in bad:
        with pytest.raises(AssertionError):
            call()
    assert ha.launch_count() == launches


@pytest.mark.parametrize('bits', [16, 4])
def test_a_run_of_tokens(bits):
    """append and attention in turn, as generation uses them: a prompt, then tokens one by one and two at a time, from one captured step"""
    g = torch.Generator().manual_seed(8)
    B, H, Hk, d, page, prompt, steps = 3, 8, 2, 128, 16, [30, 1, 17], 20
    cache = ha.PagedCache.allocate(20, page, Hk, d, bits=bits)
    table = torch.randperm(20, generator=g)[:B * 6].int().view(B, 6).cuda()
    rope = rope_table(96, 64)
    total = max(prompt) + steps
    qkv = torch.randn(B, total, H + 2 * Hk, d, generator=g).to(BF).cuda()
    held = torch.zeros(B, dtype=torch.int32, device='cuda')
    counts = torch.tensor(prompt, dtype=torch.int32, device='cuda')
    parts = lambda t: t.split([H, Hk, Hk], 2)
    q, k, v = parts(qkv[:, :max(prompt)])
    ha.paged_append(cache, k, v, table, held, counts, rope, q)
    held += counts
    # every sequence's tokens after its prompt: rows max(prompt) .. of qkv
    new = torch.empty(B, 1, H + 2 * Hk, d, dtype=BF, device='cuda')
    new.copy_(qkv[:, -1:])

    def step():
        q, k, v = parts(new)
        q = ha.paged_append(cache, k, v, table, held, rope=rope, q=q)
        held.add_(1)
        return (q,) + ha.paged_attn_func(q, cache, table, held)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    at = held.clone()
    with torch.cuda.stream(s):
        step()
        held.copy_(at)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rq, ro, rl = step()
    held.copy_(at)
    hist = [[(k[b, :prompt[b]], v[b, :prompt[b]])] for b in range(B)]
    for t in range(steps):
        new.copy_(qkv[:, max(prompt) + t:max(prompt) + t + 1])
        graph.replay()
        _, k1, v1 = parts(new)
        for b in range(B):
            hist[b].append((k1[b].clone(), v1[b].clone()))
        if t % 6 == 5 or t == 0:
            ks, vs = [], []
            for b in range(B):
                kk, vv = [torch.cat([h[j] for h in hist[b]]) for j in range(2)]
                kk = rotated32(kk, rope[:kk.shape[0]])
                ks.append(kk.to(BF).double() if bits == 16 else dequantised(kk))
                vs.append(vv.double() if bits == 16 else dequantised(vv))
            lens = [p + t + 1 for p in prompt]
            assert held.tolist() == lens
            want = reference(rq, ks, vs, lens, [1] * B, d ** -0.5)
            check(ro, rl, want, bits, BF, d, max(lens), torch.full_like(want[2], 9.0) if bits == 4 else None)
