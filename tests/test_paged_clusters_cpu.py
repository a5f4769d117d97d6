"""Which calls of attention over pages go to clusters of CTAs, as the size of the workspace tells (clusters need none)."""
import ctypes as C

import pytest
import torch

from hyperattention_b200 import _lib as L


def workspace(tokens, **over):
    p = L.PagedParams()
    for name, v in dict(dict(dtype=L.BF16, bits=16, B=1, n=1, H=32, Hk=2, d=128, pages=4, page_size=16, columns=-(-tokens // 16)), **over).items():
        setattr(p, name, v)
    return L.load().ha_paged_attn_workspace_bytes(C.byref(p))


@pytest.mark.skipif(torch.cuda.is_available(), reason='of a machine without a GPU')
def test_a_device_that_holds_no_clusters_of_16():
    """(here: one that cannot be asked) 90 tiles are six for each CTA of a cluster of 16, and too many for one of 8: they go by the list"""
    assert workspace(80 * 64) == 0                          # ten each for eight
    assert workspace(90 * 64) > 0
    assert workspace(90 * 128, bits=4) > 0


@pytest.mark.gpu
def test_a_device_that_holds_them():
    assert workspace(90 * 64) == 0 and workspace(96 * 64) == 0 and workspace(97 * 64) > 0
