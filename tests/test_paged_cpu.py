"""The paged key/value cache without a GPU: what the handle and the C entry points refuse (no kernel is launched), and the 4-bit row format."""
import ctypes as C
import math
import os

import pytest
import torch

import hyperattention_b200 as ha
from hyperattention_b200 import _lib as L


@pytest.fixture(scope='module')
def lib():
    if not os.path.exists(L.LIB_PATH):
        import __graft_entry__
        __graft_entry__.build()
    return L.load()


def test_struct_layout_matches_header():
    assert C.sizeof(L.PagedParams) == 16 * 4 + 3 * 8 + 9 * 8 + 5 * 8 + 5 * 8 + 5 * 8 + 5 * 8 + 5 * 8


def _params(**over):
    p = L.PagedParams()
    dummy = C.c_void_p(256)
    vals = dict(dtype=L.BF16, bits=16, B=2, n=1, H=8, Hk=2, d=128, pages=4, page_size=16, columns=3, scale=0.1,
                q=dummy, k=dummy, v=dummy, q_sb=1024, q_sn=1024, q_sh=128, k_sb=256, k_sn=256, k_sh=128, v_sb=256, v_sn=256, v_sh=128,
                k_pages=dummy, v_pages=dummy, page_sp=4096, page_sh=2048, page_st=128, k_scales=dummy, v_scales=dummy, scale_sp=128, scale_sh=64,
                scale_st=4, table=dummy, table_sb=3, lengths=dummy, q_out=dummy, k_out=dummy, v_out=dummy, o=dummy, lse=dummy, rows=10,
                workspace=dummy, workspace_bytes=1)
    vals.update(over)
    for name, v in vals.items():
        setattr(p, name, v)
    return p


BAD = [(dict(dtype=L.FP32), -2), (dict(dtype=9), -2), (dict(bits=8), -1), (dict(d=96), -1), (dict(d=0), -1), (dict(B=-1), -1), (dict(n=-1), -1),
       (dict(Hk=0), -1), (dict(H=7), -1), (dict(pages=-1), -1), (dict(page_size=0), -1), (dict(columns=-1), -1),
       (dict(columns=1 << 20, page_size=1 << 20), -5), (dict(columns=2 ** 31 - 1, page_size=1), -5), (dict(columns=1, page_size=2 ** 31 - 1), -5), (dict(lengths=None), -1), (dict(table=None), -1), (dict(k_pages=None), -1), (dict(v_pages=None), -1),
       (dict(k_pages=264), -1), (dict(page_st=100), -1), (dict(page_sp=-4096), -1), (dict(bits=4, k_scales=None), -1), (dict(bits=4, v_scales=260), -1),
       (dict(bits=4, scale_st=2), -1), (dict(bits=4, page_st=72), -1)]


@pytest.mark.parametrize('over,want', BAD, ids=[str(b[0]) for b in BAD])
def test_entry_points_refuse(lib, over, want):
    launches = lib.ha_launch_count()
    for fn in (lib.ha_paged_append, lib.ha_paged_attn, lib.ha_paged_gather):
        assert fn(C.byref(_params(**over)), None) == want
    assert lib.ha_launch_count() == launches


def test_entry_points_refuse_their_own(lib):
    launches = lib.ha_launch_count()
    for over in (dict(k=None), dict(v=None), dict(q=None), dict(q_out=None), dict(k_out=264), dict(rope=256, rot=3), dict(rope=256, rot=130),
                 dict(rope=256, rot=64, rope_dtype=L.FP16), dict(rope=256, rot=64, rope_rows=-1)):
        assert lib.ha_paged_append(C.byref(_params(**over)), None) == -1, over
    for over in (dict(q=None), dict(o=None), dict(lse=None), dict(q=264), dict(q_sh=100), dict(H=0), dict(scale=0.0), dict(scale=math.nan),
                 dict(scale=math.inf), dict(scale=-math.inf), dict(scale=1e-38)):
        assert lib.ha_paged_attn(C.byref(_params(**over)), None) == -1, over
    assert lib.ha_paged_attn(C.byref(_params(columns=4000)), None) == -3                        # workspace too small
    assert lib.ha_paged_attn(C.byref(_params(workspace=None, columns=4000)), None) == -3
    for over in (dict(rows=-1), dict(k_out=None), dict(v_out=264)):
        assert lib.ha_paged_gather(C.byref(_params(**over)), None) == -1, over
    for fn in (lib.ha_paged_append, lib.ha_paged_attn, lib.ha_paged_gather):
        assert fn(None, None) == -1
        assert fn(C.byref(_params(B=0)), None) == 0                                             # nothing to do
    assert lib.ha_launch_count() == launches
    # workspace: two parts of 16 rows a CTA; none where a cluster shares an item
    one = lib.ha_paged_attn_workspace_bytes(C.byref(_params(B=1, Hk=1, columns=4000)))
    assert one == 256 + 296 * (16 + 2 * 16 * (128 * 4 + 8))
    assert lib.ha_paged_attn_workspace_bytes(C.byref(_params(B=0))) == 0 and lib.ha_paged_attn_workspace_bytes(C.byref(_params())) == 0
    assert lib.ha_paged_attn_workspace_bytes(C.byref(_params(d=96))) == -1


def test_handle_refuses():
    t = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt)
    codes, scales = t(3, 2, 16, 64, dt=torch.uint8), t(3, 2, 16, 2, 2, dt=torch.float16)
    ha.PagedCache(t(3, 2, 16, 128), t(3, 2, 16, 128))
    c = ha.PagedCache(codes, codes.clone(), scales, scales.clone())
    assert (c.bits, c.head_dim, c.dtype, c.page_size, c.kv_heads, c.pages) == (4, 128, torch.bfloat16, 16, 2, 3)
    for bad in ((t(3, 2, 16, 96), t(3, 2, 16, 96)), (t(3, 2, 16, 128), t(3, 2, 8, 128)), (t(3, 2, 16, 128), t(3, 2, 16, 128, dt=torch.float16)),
                (t(3, 2, 16, 64, dt=torch.float32), t(3, 2, 16, 64, dt=torch.float32)), (t(3, 2, 128, 16).transpose(2, 3), t(3, 2, 128, 16).transpose(2, 3)),
                (t(3, 2, 16, 132)[..., :128], t(3, 2, 16, 132)[..., :128]), (t(3, 2, 16, 128), t(3, 16, 2, 128).transpose(1, 2)),
                (codes, codes, scales, None), (codes, codes, scales[..., :1], scales[..., :1]), (codes, codes, scales.bfloat16(), scales.bfloat16()),
                (codes, codes, scales, scales, torch.float32), (t(3, 2, 16, 128), t(3, 2, 16, 128), None, None, torch.float16)):
        with pytest.raises(AssertionError):
            ha.PagedCache(*bad)
    with pytest.raises(AssertionError):
        ha.PagedCache.allocate(3, 16, 2, 128, bits=8, device='cpu')
    with pytest.raises(AssertionError):
        ha.PagedCache.allocate(3, 16, 2, 80, device='cpu')


def test_operators_refuse_cpu_tensors():
    c = ha.PagedCache.allocate(3, 16, 2, 64, device='cpu')
    k, table, lengths = torch.zeros(1, 1, 2, 64, dtype=torch.bfloat16), torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: ha.paged_append(c, k, k, table, lengths), lambda: ha.paged_attn_func(k, c, table, lengths),
                 lambda: ha.paged_gather(c, table, lengths, 4)):
        with pytest.raises(AssertionError, match='CUDA'):
            call()


@pytest.mark.parametrize('d', [64, 128])
def test_values_of_codes(d):
    """values() against the format spelled out element by element"""
    g = torch.Generator().manual_seed(0)
    codes = torch.randint(0, 256, (2, 1, 3, d // 2), generator=g, dtype=torch.uint8)
    scales = torch.randn(2, 1, 3, d // 64, 2, generator=g).half()
    got, _ = ha.PagedCache(codes, codes, scales, scales).values()
    for at in ((0, 0, 0), (1, 0, 2)):
        for e in range(d):
            word = (e % 64 // 8) * (d // 64) + e // 64
            byte = int(codes[at][word * 4 + e % 8 // 2])
            s, m = scales[at][e // 64].float()
            assert float(got[at][e]) == float(((byte >> (4 * (e % 2))) & 15) * s + m)
