"""Attention over pages by the list of tiles, whose parts a second kernel joins: the tests of test_gpu_paged.py, most of whose contexts go to clusters, once more with
tables as wide as a server's (65536 positions and more, which no cluster takes).  Tolerances are those of that file."""
import ctypes as C
import itertools
import math

import pytest
import torch

import hyperattention_b200 as ha
import test_gpu_paged as paged
from hyperattention_b200 import _lib as L

BF, HF = torch.bfloat16, torch.float16
MOST = 65536
gpu = pytest.mark.gpu


@pytest.fixture
def wide(monkeypatch):
    make = paged.make_cache

    def make_wide(rows_k, rows_v, page, *args, **kw):
        cache, table, ks, vs = make(rows_k, rows_v, page, *args, **kw)
        more = max(-(-MOST // page) - table.shape[1], 0)
        return cache, torch.cat([table, torch.full((table.shape[0], more), -9, dtype=torch.int32, device='cuda')], 1), ks, vs

    monkeypatch.setattr(paged, 'make_cache', make_wide)


def params(**over):
    p = L.PagedParams()
    for name, v in dict(dict(dtype=L.BF16, bits=16, B=1, n=1, H=8, Hk=2, d=128, pages=4, page_size=16, columns=MOST // 16, scale=0.1), **over).items():
        setattr(p, name, v)
    return p


def test_wide_tables_go_by_the_list():
    """(a workspace is what the list needs and clusters do not)"""
    lib = L.load()
    for bits, d, B, n, (H, Hk), page in itertools.product((16, 4), (64, 128), (1, 3, 64, 500), (1, 2, 8, 16), ((1, 1), (4, 2), (16, 1), (32, 2), (40, 2)), (1, 16, 1000)):
        p = params(bits=bits, d=d, B=B, n=n, H=H, Hk=Hk, page_size=page, columns=-(-MOST // page))
        assert lib.ha_paged_attn_workspace_bytes(C.byref(p)) > 0


@gpu
@pytest.mark.parametrize('bits', [16, 4])
@pytest.mark.parametrize('dtype', [BF, HF])
@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('H,Hk', [(1, 1), (4, 4), (6, 2), (8, 1), (16, 1), (32, 2), (34, 2), (40, 2)])
def test_heads_and_types(wide, bits, dtype, d, H, Hk):
    paged.test_attention_heads_and_types(bits, dtype, d, H, Hk)


@gpu
@pytest.mark.parametrize('bits', [16, 4])
@pytest.mark.parametrize('dtype', [BF, HF])
@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('H,Hk,n', [(16, 1, 1), (32, 2, 1), (2, 2, 1), (6, 2, 4), (32, 2, 3)])
def test_several_tiles_of_a_part(wide, bits, dtype, d, H, Hk, n):
    """contexts of hundreds of tiles beside short and empty ones: CTAs that hold an item's middle, its end, several items"""
    paged.attend_case(bits, dtype, d, H, Hk, 64, [9000, n, 20011, 0, 64, 5000], n=n)
    paged.attend_case(bits, dtype, d, H, Hk, 48, [40000], n=n)


@gpu
@pytest.mark.parametrize('bits', [16, 4])
@pytest.mark.parametrize('page', [1, 7, 16, 64, 100, 1000])
def test_page_sizes(wide, bits, page):
    paged.test_attention_page_sizes(bits, page)


@gpu
@pytest.mark.parametrize('bits', [16, 4])
@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('length', [1, 2, 63, 64, 65, 127, 128, 129, 255, 256, 257, 513, 4097, 20011])
def test_lengths(wide, bits, d, length):
    paged.test_attention_lengths(bits, d, length)


@gpu
@pytest.mark.parametrize('bits', [16, 4])
@pytest.mark.parametrize('n', [2, 3, 8])
def test_several_tokens(wide, bits, n):
    paged.test_attention_several_tokens(bits, n)


@gpu
@pytest.mark.parametrize('bits', [16, 4])
@pytest.mark.parametrize('dtype', [BF, HF])
@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('H,Hk,n', [(1, 1, 16), (2, 2, 5), (6, 2, 4), (8, 1, 3), (16, 4, 9), (5, 1, 17)])
def test_tokens_share_an_item(wide, bits, dtype, d, H, Hk, n):
    paged.test_attention_tokens_share_an_item(bits, dtype, d, H, Hk, n)


@gpu
@pytest.mark.parametrize('bits', [16, 4])
@pytest.mark.parametrize('what', [math.nan, math.inf])
@pytest.mark.parametrize('d', [64, 128])
def test_tokens_of_an_item_keep_apart(wide, bits, what, d):
    paged.test_attention_tokens_of_an_item_keep_apart(bits, what, d)


@gpu
@pytest.mark.parametrize('dtype', [BF, HF])
@pytest.mark.parametrize('d', [64, 128])
@pytest.mark.parametrize('n', [1, 4, 16])
def test_infinite_values(wide, dtype, d, n):
    paged.test_attention_infinite_values(dtype, d, n)


@gpu
@pytest.mark.parametrize('bits', [16, 4])
def test_the_rest(wide, bits):
    paged.test_attention_large_and_small_scores(bits)
    paged.test_attention_values_that_are_no_numbers(bits)
    paged.test_attention_query_strides(bits, 'view')
    if bits == 16:
        paged.test_attention_weights_over_a_sink()               # (both widths)
        paged.test_attention_no_numbers_in_a_whole_warp()
        paged.test_attention_token_major_pages()
        paged.test_shared_pages()


@gpu
@pytest.mark.parametrize('bits', [16, 4])
def test_repeats_and_streams(wide, bits):
    paged.test_attention_repeats_and_streams(bits)


@gpu
@pytest.mark.parametrize('bits', [16, 4])
@pytest.mark.parametrize('columns', ['tight', 'wide'])
def test_a_graph_whose_table_changes(request, bits, columns):
    """pages that move between replays, sequences that change places, lengths that grow and shrink"""
    if columns == 'wide':
        request.getfixturevalue('wide')
    g = torch.Generator().manual_seed(9)
    lens, d, page = [700, 64, 3000], 128, 16
    rk, rv = [[torch.randn(l, 2, d, generator=g) for l in lens] for _ in 'kv']
    cache, table, ks, vs = paged.make_cache(rk, rv, page, bits, BF, g, spare=200)
    q = torch.randn(3, 1, 32, d, generator=g).to(BF).cuda()
    length = torch.tensor(lens, dtype=torch.int32, device='cuda')
    graph = torch.cuda.CUDAGraph()
    ha.paged_attn_func(q, cache, table, length)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        o, lse = ha.paged_attn_func(q, cache, table, length)

    def replayed(now):
        graph.replay()
        want = paged.reference(q, ks, vs, now, [1, 1, 1], d ** -0.5)
        paged.check(o, lse, want, bits, BF, d, max(now), torch.full_like(want[2], 8.0) if bits == 4 else None)

    replayed(lens)
    # half of the pages go elsewhere; where they were, nothing is a number
    used = set(int(p) for b, l in enumerate(lens) for p in table[b, :-(-l // page)])
    free = [p for p in range(cache.pages) if p not in used]
    for b, l in enumerate(lens):
        for c in range(0, -(-l // page), 2):
            if not free:
                break
            old, new = int(table[b, c]), free.pop()
            for t in (cache.k, cache.v, cache.k_scales, cache.v_scales):
                if t is not None:
                    t[new].copy_(t[old])
            for t in (cache.k_scales, cache.v_scales) if bits == 4 else (cache.k, cache.v):
                t[old].fill_(math.nan)
            table[b, c] = new
    replayed(lens)
    # the first and the last sequence change places
    table[[0, 2]] = table[[2, 0]]
    ks[0], ks[2], vs[0], vs[2] = ks[2], ks[0], vs[2], vs[0]
    length.copy_(torch.tensor(lens[::-1], dtype=torch.int32))
    replayed(lens[::-1])
    length.copy_(torch.tensor([2999, 0, 1], dtype=torch.int32))
    replayed([2999, 0, 1])


@gpu
@pytest.mark.parametrize('bits', [16, 4])
@pytest.mark.parametrize('length', [200, 30000])
def test_c_entry_points(bits, length):
    """the C functions as a C program calls them, without maps kept from an earlier call: the bits of the Python operators"""
    lib, g, i32 = L.load(), torch.Generator().manual_seed(1), dict(dtype=torch.int32, device='cuda')
    H, Hk, d, page, n = 8, 2, 128, 16, 3
    pages = -(-(length + n) // page)
    caches = [ha.PagedCache.allocate(pages, page, Hk, d, bits=bits) for _ in range(2)]
    table = torch.randperm(pages, generator=g).int().cuda()[None]
    old = torch.randn(2, 1, length, Hk, d, generator=g).to(BF).cuda()
    q, k, v = [torch.randn(1, n, h, d, generator=g).to(BF).cuda() for h in (H, Hk, Hk)]
    rope = paged.rope_table(length + n, 64)
    for c in caches:
        ha.paged_append(c, old[0], old[1], table, torch.zeros(1, **i32), rope=rope)
    held = torch.full((1,), length, **i32)
    turned = ha.paged_append(caches[0], k, v, table, held, rope=rope, q=q)
    want = ha.paged_attn_func(turned, caches[0], table, held + n)
    dense = ha.paged_gather(caches[0], table, held + n, length + n)

    c = caches[1]
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    status = torch.zeros(1, **i32)
    total = held + n
    out = {name: torch.full_like(t, math.nan) for name, t in dict(q_out=turned, o=want[0], lse=want[1], k_out=dense[0], v_out=dense[1]).items()}
    over = dict(bits=bits, n=n, H=H, Hk=Hk, d=d, pages=pages, page_size=page, columns=table.shape[1], rot=64, rope_rows=rope.shape[0], rope_dtype=L.FP32,
                rows=length + n, scale=d ** -0.5, q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), k_pages=c.k.data_ptr(), v_pages=c.v.data_ptr(),
                page_sp=c.k.stride(0), page_sh=c.k.stride(1), page_st=c.k.stride(2), table=table.data_ptr(), table_sb=table.shape[1], lengths=held.data_ptr(),
                rope=rope.data_ptr(), q_out=out['q_out'].data_ptr(), status=status.data_ptr())
    for name, t in dict(q=q, k=k, v=v).items():
        over.update({f'{name}_sb': t.stride(0), f'{name}_sn': t.stride(1), f'{name}_sh': t.stride(2)})
    if bits == 4:
        over.update(k_scales=c.k_scales.data_ptr(), v_scales=c.v_scales.data_ptr(), scale_sp=c.k_scales.stride(0), scale_sh=c.k_scales.stride(1), scale_st=c.k_scales.stride(2))
    assert lib.ha_paged_append(C.byref(params(**over)), stream) == 0
    over.update(lengths=total.data_ptr(), q=out['q_out'].data_ptr(), o=out['o'].data_ptr(), lse=out['lse'].data_ptr(), k_out=out['k_out'].data_ptr(),
                v_out=out['v_out'].data_ptr())
    size = lib.ha_paged_attn_workspace_bytes(C.byref(params(**over)))
    assert (size > 0) == (length == 30000)
    ws = torch.empty(max(size, 1), dtype=torch.uint8, device='cuda')
    over.update(workspace=ws.data_ptr(), workspace_bytes=size)
    p = params(**over)
    assert not p.maps and lib.ha_paged_attn(C.byref(p), stream) == 0
    assert lib.ha_paged_gather(C.byref(p), stream) == 0
    torch.cuda.synchronize()
    assert int(status) == 0
    assert torch.equal(out['q_out'], turned) and torch.equal(out['o'], want[0]) and torch.equal(out['lse'], want[1])
    assert torch.equal(out['k_out'], dense[0]) and torch.equal(out['v_out'], dense[1])
