"""Generation with a paged key/value cache: rows are appended (position rotation and, for a cache in 4 bits, coding on the way), a sequence's last
tokens attend to its pages, and a context is read back as dense tensors for the prompt's attention.  No counterpart in the reference, whose
attention covers prompts only.

A cache is a pool of pages; a page holds ``page_size`` token rows of every K/V head.  A table names the pages of each sequence in order: position t of
sequence b lies in page ``table[b, t // page_size]``, row ``t % page_size``.  Sequences may share pages that nobody appends to.

    cache = PagedCache.allocate(pages, page_size, kv_heads, head_dim, bits=16)
    q = paged_append(cache, k, v, table, held, rope=rope, q=q)            # the new tokens' rows, at positions held[b] ..
    o, lse = paged_attn_func(q, cache, table, held + n)

All tensors lie on one device; everything is enqueued on its current stream, nothing synchronises, and calls can be captured into CUDA graphs (lengths
and tables are read on the device at every replay).  A position beyond the table or the rotation's rows, or a page that does not exist, is
neither written nor read and is reported by the next call into the library (or ``check_device_status()``), as a device-side timeout is.  The
operators have no gradient.
"""
import ctypes as C
import os

import torch
from torch.autograd import forward_ad

from . import _lib as L
from . import ops

GROUP = 64          # elements of a row that share a step and an offset in a 4-bit cache
_ROWS = (torch.bfloat16, torch.float16)
_EXT = None


def _ext():
    """The operators' host side (csrc/paged_ext.cpp: checks, allocations and the call into the library), loaded once."""
    global _EXT
    if _EXT is None:
        if not os.path.exists(os.path.join(os.path.dirname(__file__), '_paged_ext.so')):
            raise RuntimeError('_paged_ext.so is missing: build it with `python hyperattention_b200/csrc/build.py` (there is no fallback implementation)')
        from . import _paged_ext
        lib = L.load()
        _paged_ext.init(*[C.cast(getattr(lib, 'ha_paged_' + f), C.c_void_p).value for f in ('append', 'attn', 'gather', 'maps', 'attn_workspace_bytes')])
        _EXT = _paged_ext
    return _EXT


class PagedCache:
    """The pages of one layer.

    16 bits: ``k``, ``v`` [pages, kv_heads, page_size, head_dim], bf16 or fp16.
    4 bits:  ``k``, ``v`` uint8 [pages, kv_heads, page_size, head_dim / 2] and ``k_scales``, ``v_scales`` fp16
             [pages, kv_heads, page_size, head_dim / 64, 2]; ``dtype`` is the type of the rows that go in and come out.  Each group of 64
             elements is held as codes 0 .. 15 with a step and the value of code 0: what ``values()`` gives.

    The tensors may be views of a larger pool (any strides that K and V share; rows contiguous and on 16-byte boundaries), and belong to the caller:
    the handle checks them once and keeps them."""

    def __init__(self, k, v, k_scales=None, v_scales=None, dtype=None):
        self._tensors = (k, v) if k_scales is None and v_scales is None else (k, v, k_scales, v_scales)
        self.bits = 16 if k_scales is None else 4
        assert (k_scales is None) == (v_scales is None), 'a 4-bit cache has scales of both K and V'
        assert k.dim() == 4 and k.shape == v.shape and k.dtype == v.dtype and k.device == v.device, 'K and V pages must be alike'
        assert k.stride() == v.stride(), 'K and V pages must have the same strides'
        assert k.stride(-1) == 1, 'rows of a page must be contiguous'
        if self.bits == 16:
            self.dtype = k.dtype
            assert dtype is None or dtype == k.dtype, 'a 16-bit cache holds rows of its own type'
            self.head_dim = k.shape[3]
        else:
            self.dtype = torch.bfloat16 if dtype is None else dtype
            assert k.dtype == torch.uint8, 'codes must be uint8'
            self.head_dim = 2 * k.shape[3]
            want = k.shape[:3] + (self.head_dim // GROUP, 2)
            assert k_scales.shape == want and v_scales.shape == want, f'scales must have shape {tuple(want)}'
            assert k_scales.dtype == torch.float16 and v_scales.dtype == torch.float16, 'scales must be fp16'
            assert k_scales.device == k.device and v_scales.device == k.device, 'all tensors must be on one device'
            assert k_scales.stride() == v_scales.stride() and k_scales.stride()[3:] == (2, 1), 'scales must have the same strides, rows contiguous'
        assert self.dtype in _ROWS, 'Only support fp16 and bf16'
        assert self.head_dim in (64, 128), 'head dimensions 64 and 128 are supported'
        self.pages, self.kv_heads, self.page_size = k.shape[:3]
        assert self.page_size >= 1 and self.kv_heads >= 1
        unit, sc = 16 // k.element_size(), self.head_dim // GROUP * 2
        assert all(s % unit == 0 for s in k.stride()[:3]) and k.data_ptr() % 16 == 0 and v.data_ptr() % 16 == 0, 'rows must lie on 16-byte boundaries'
        if self.bits == 4:
            assert all(s % sc == 0 for s in k_scales.stride()[:3]) and k_scales.data_ptr() % (2 * sc) == 0 and v_scales.data_ptr() % (2 * sc) == 0, \
                'scales of a row must lie on a boundary of their size'
        self.device = k.device
        p = L.PagedParams()
        p.dtype, p.bits, p.Hk, p.d, p.pages, p.page_size = ops._DT[self.dtype], self.bits, self.kv_heads, self.head_dim, self.pages, self.page_size
        p.page_sp, p.page_sh, p.page_st = k.stride()[:3]
        if self.bits == 4:
            p.scale_sp, p.scale_sh, p.scale_st = k_scales.stride()[:3]
        for name, t in zip(('k_pages', 'v_pages', 'k_scales', 'v_scales'), self._tensors):
            setattr(p, name, t.data_ptr())
        self._params = p                 # the parameters of a call that the cache decides
        self._handle = None

    def _open(self):
        """What the operators' host side keeps of the cache: made at the first call."""
        host_word = 0
        if self.device.type == 'cuda':
            ops._status_words(self.device)
            self._params.status, self._params.status_host = ops._STATUS_RAW[self.device.index][:2]
            host_word = self._params.status_host
        self._handle = _ext().open(bytes(self._params), host_word, *self._tensors)
        return self._handle

    k = property(lambda self: self._tensors[0])
    v = property(lambda self: self._tensors[1])
    k_scales = property(lambda self: self._tensors[2] if self.bits == 4 else None)
    v_scales = property(lambda self: self._tensors[3] if self.bits == 4 else None)

    @classmethod
    def allocate(cls, pages, page_size, kv_heads, head_dim, dtype=torch.bfloat16, bits=16, device='cuda'):
        """An empty cache.  The rows are not initialised: nothing reads a row before it was appended."""
        assert bits in (16, 4), 'a cache is held in 16 or 4 bits'
        assert head_dim in (64, 128), 'head dimensions 64 and 128 are supported'
        shape = (pages, kv_heads, page_size)
        if bits == 16:
            return cls(*[torch.empty(*shape, head_dim, dtype=dtype, device=device) for _ in 'kv'])
        return cls(*[torch.empty(*shape, head_dim // 2, dtype=torch.uint8, device=device) for _ in 'kv'],
                   *[torch.empty(*shape, head_dim // GROUP, 2, dtype=torch.float16, device=device) for _ in 'kv'], dtype=dtype)

    def values(self):
        """(k, v) as fp32 tensors [pages, kv_heads, page_size, head_dim], whatever the pages hold (plain torch; for looking, not for speed)."""
        if self.bits == 16:
            return self.k.float(), self.v.float()
        out = []
        for codes, scales in ((self.k, self.k_scales), (self.v, self.v_scales)):
            q = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).unflatten(-1, (8, -1, 8)).transpose(-3, -2).flatten(-2).float()
            out.append((q * scales[..., :1].float() + scales[..., 1:].float()).flatten(-2))
        return tuple(out)


_transforms = torch._C._are_functorch_transforms_active


def _handle(cache):
    # forward-mode differentiation and function transforms would lose their tangents without a word
    assert forward_ad._current_level < 0 and not _transforms(), 'the operators of the paged cache have no gradient: call them under torch.no_grad()'
    return cache._handle or cache._open()


def _settle(r, name, cache):
    """What an operator's host side answers in the place of outputs: a status, or NotImplemented where an earlier launch has reported a failure, which is raised
    here, as at every call into the library (and gone when it has been raised elsewhere meanwhile)."""
    if r is NotImplemented:
        ops._raise_if_failed(*ops._status_words(cache.device))
    else:
        L.check(r, 'ha_paged_' + name)


def paged_append(cache, k, v, table, lengths, counts=None, rope=None, q=None, return_keys=False):
    """Writes the rows k, v [B, n, kv_heads, head_dim] of n new tokens a sequence to their pages.

    lengths  int32 [B]: tokens that each sequence holds already; row i goes to position lengths[b] + i
    counts   int32 [B] or None: rows of each sequence that are tokens; the others (padding) are not written
    rope     [positions, rot / 2, 2] cosines and sines by position, fp32 or the cache's type, or None: the first rot elements of every key (and query) are
             rotated in pairs (2j, 2j + 1), in 32 bits
    q        [B, n, heads, head_dim] or None: queries to rotate alike

    Returns the rotated queries [B, n, heads, head_dim] (None without q); with return_keys, (queries, rotated keys [B, n, kv_heads, head_dim]): what the
    prompt's own attention takes.  Padding rows of both are zero.  Two rows of one call must not go to the same slot."""
    r = (_EXT or _ext()).append(_handle(cache), k, v, table, lengths, counts, rope, q, return_keys)
    if r.__class__ is int or r is NotImplemented:
        _settle(r, 'append', cache)
        return paged_append(cache, k, v, table, lengths, counts, rope, q, return_keys)
    return r


def paged_attn_func(q, cache, table, lengths, counts=None, softmax_scale=None):
    """Attention of the last n tokens of every sequence over its pages: q [B, n, heads, head_dim] -> o [B, n, heads, head_dim], lse fp32 [B, heads, n].

    lengths  int32 [B]: tokens that each sequence holds, the new ones among them
    counts   int32 [B] or None: rows of q that are tokens of the sequence, n of each without it
    softmax_scale  head_dim ** -0.5 without it; 0 is refused

    Row i < counts[b] sees positions 0 .. lengths[b] - counts[b] + i.  A row that sees none, and padding rows, have o = 0 and lse = -inf.  Consecutive
    query heads share a K/V head.  Keys are read once for 16 query rows of a K/V head, those of neighbouring tokens where a token has fewer, and again
    for the next 16: made for one to a few tokens a sequence; prompts belong to HyperAttention or flash_attn_func.  Over a cache in 4 bits,
    queries of 1e34 and more are not told from infinite ones."""
    r = (_EXT or _ext()).attn(_handle(cache), q, table, lengths, counts, float(cache.head_dim ** -0.5 if softmax_scale is None else softmax_scale))
    if r.__class__ is int or r is NotImplemented:
        _settle(r, 'attn', cache)
        return paged_attn_func(q, cache, table, lengths, counts, softmax_scale)
    return r


def paged_gather(cache, table, lengths, rows):
    """Positions 0 .. rows - 1 of every sequence as dense (k, v) [B, kv_heads, rows, head_dim] in the cache's type, zero from lengths[b] (int32 [B]) on: the
    layout that HyperAttention takes."""
    r = (_EXT or _ext()).gather(_handle(cache), table, lengths, int(rows))
    if r.__class__ is int or r is NotImplemented:
        _settle(r, 'gather', cache)
        return paged_gather(cache, table, lengths, rows)
    return r
