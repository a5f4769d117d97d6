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

import torch

from . import _lib as L
from . import ops

GROUP = 64          # elements of a row that share a step and an offset in a 4-bit cache
_ROWS = (torch.bfloat16, torch.float16)


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
        self._raw = bytes(p)             # the parameters of a call that the cache decides
        self._at = [t.data_ptr() for t in self._tensors]
        self._maps = None                # what the attention kernel keeps about 16-bit pages
        self._plans = {}                 # parameters of calls by their tensors' shapes and strides (bounded); no pointers but the cache's own

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

    def _check_place(self):
        assert [t.data_ptr() for t in self._tensors] == self._at, 'the pages have moved: make a new PagedCache'

    def _plan(self, key, make):
        """Parameters of a call whose tensors have the shapes, strides and types of `key`: checked and filled in once."""
        plan = self._plans.get(key)
        if plan is None:
            p = L.PagedParams.from_buffer_copy(self._raw)
            rest = make(p)
            if len(self._plans) >= 256:
                self._plans.clear()
            plan = self._plans[key] = (bytes(p), rest)
        return plan


def _form(t):
    return None if t is None else (t.shape, t.stride(), t.dtype, t.get_device())


# (an allocation of known strides costs a third less host time than torch.empty, and these calls are that time where the batch is small)
_new = torch.empty_strided


def _dense(*shape):
    """Sizes and strides of a contiguous tensor."""
    strides, n = [], 1
    for s in reversed(shape):
        strides.append(n)
        n *= max(s, 1)
    return shape, tuple(reversed(strides))


def _places(p, cache, table, lengths, counts, B):
    """Checks the table and the lengths of a call, and fills in their sizes."""
    ops._cuda(cache.k)
    dev = cache.device
    assert table.dim() == 2 and table.shape[0] == B and table.dtype == torch.int32 and (table.stride(1) == 1 or table.shape[1] <= 1), \
        'table must be int32 [batch, columns], rows contiguous'
    assert lengths.shape == (B,) and lengths.dtype == torch.int32 and lengths.is_contiguous(), 'lengths must be contiguous int32 [batch]'
    assert table.device == dev and lengths.device == dev, 'all tensors must be on one device'
    if counts is not None:
        assert counts.shape == (B,) and counts.dtype == torch.int32 and counts.is_contiguous() and counts.device == dev, \
            'counts must be contiguous int32 [batch]'
    p.B, p.columns, p.table_sb = B, table.shape[1], table.stride(0)


def _rows(cache, t, B, n, heads, what):
    assert t.dim() == 4 and t.shape == (B, n, heads, cache.head_dim), f'{what} must be [batch, tokens, heads, head_dim] with the head_dim of the cache'
    assert t.dtype == cache.dtype and t.device == cache.device, f'{what} must have the type and device of the cache'


def _no_grad(*ts):
    assert not ops._wants_grad(*ts), 'the operators of the paged cache have no gradient: call them under torch.no_grad()'


def paged_append(cache, k, v, table, lengths, counts=None, rope=None, q=None, return_keys=False):
    """Writes the rows k, v [B, n, kv_heads, head_dim] of n new tokens a sequence to their pages.

    lengths  int32 [B]: tokens that each sequence holds already; row i goes to position lengths[b] + i
    counts   int32 [B] or None: rows of each sequence that are tokens; the others (padding) are not written
    rope     [positions, rot / 2, 2] cosines and sines by position, fp32 or the cache's type, or None: the first rot elements of every key (and query) are
             rotated in pairs (2j, 2j + 1), in 32 bits
    q        [B, n, heads, head_dim] or None: queries to rotate alike

    Returns the rotated queries [B, n, heads, head_dim] (None without q); with return_keys, (queries, rotated keys [B, n, kv_heads, head_dim]): what the
    prompt's own attention takes.  Padding rows of both are zero.  Two rows of one call must not go to the same slot."""
    # rows that are not contiguous are copied, as in HyperAttention
    k, v, q = [t if t is None or t.dim() == 0 or t.stride(-1) == 1 else t.contiguous() for t in (k, v, q)]
    _no_grad(k, v) if q is None else _no_grad(k, v, q)

    def make(p):
        assert k.dim() == 4, 'k must be [batch, tokens, heads, head_dim]'
        B, p.n = k.shape[:2]
        _places(p, cache, table, lengths, counts, B)
        _rows(cache, k, B, p.n, cache.kv_heads, 'k')
        _rows(cache, v, B, p.n, cache.kv_heads, 'v')
        p.k_sb, p.k_sn, p.k_sh, _ = k.stride()
        p.v_sb, p.v_sn, p.v_sh, _ = v.stride()
        if q is not None:
            assert q.dim() == 4 and q.shape[2] % cache.kv_heads == 0, 'query heads must be a multiple of the key/value heads'
            _rows(cache, q, B, p.n, q.shape[2], 'q')
            p.H = q.shape[2]
            p.q_sb, p.q_sn, p.q_sh, _ = q.stride()
        if rope is not None:
            assert rope.dim() == 3 and rope.shape[2] == 2 and rope.is_contiguous() and rope.device == cache.device, 'rope must be contiguous [positions, rot / 2, 2]'
            assert rope.dtype in (torch.float32, cache.dtype) and 2 * rope.shape[1] <= cache.head_dim, \
                'rope must be fp32 or of the cache\'s type, for at most head_dim elements'
            p.rot, p.rope_rows, p.rope_dtype = 2 * rope.shape[1], rope.shape[0], ops._DT[rope.dtype]
        return _dense(*k.shape), None if q is None else _dense(*q.shape)

    cache._check_place()
    raw, (k_form, q_form) = cache._plan(('append', _form(k), _form(v), _form(q), _form(table), _form(lengths), _form(counts), _form(rope)), make)
    p = L.PagedParams.from_buffer_copy(raw)
    ops._set_status(p, cache.device)
    p.k, p.v, p.table, p.lengths = k.data_ptr(), v.data_ptr(), table.data_ptr(), lengths.data_ptr()
    q_out = k_out = None
    if counts is not None:
        p.counts = counts.data_ptr()
    if rope is not None:
        p.rope = rope.data_ptr()
    if q is not None:
        q_out = _new(*q_form, dtype=cache.dtype, device=cache.device)
        p.q, p.q_out = q.data_ptr(), q_out.data_ptr()
    if return_keys:
        k_out = _new(*k_form, dtype=cache.dtype, device=cache.device)
        p.k_out = k_out.data_ptr()
    L.check(ops._call(L.load().ha_paged_append, cache.device, C.byref(p)), 'ha_paged_append')
    return (q_out, k_out) if return_keys else q_out


def paged_attn_func(q, cache, table, lengths, counts=None, softmax_scale=None):
    """Attention of the last n tokens of every sequence over its pages: q [B, n, heads, head_dim] -> o [B, n, heads, head_dim], lse fp32 [B, heads, n].

    lengths  int32 [B]: tokens that each sequence holds, the new ones among them
    counts   int32 [B] or None: rows of q that are tokens of the sequence, n of each without it

    Row i < counts[b] sees positions 0 .. lengths[b] - counts[b] + i.  A row that sees none, and padding rows, have o = 0 and lse = -inf.  Consecutive
    query heads share a K/V head.  Every token reads the sequence's keys again (from the L2 cache where they fit): made for one to a few
    tokens a sequence; prompts belong to HyperAttention or flash_attn_func."""
    _no_grad(q)
    if q.dim() == 4 and (q.stride(3) != 1 or (q.data_ptr() | 2 * (q.stride(0) | q.stride(1) | q.stride(2))) % 16):
        q = q.clone(memory_format=torch.contiguous_format)             # rows that the kernel's 16-byte loads cannot read
    scale = float(softmax_scale or cache.head_dim ** -0.5)

    def make(p):
        assert q.dim() == 4 and q.shape[2] % cache.kv_heads == 0 and q.shape[2] > 0, 'q must be [batch, tokens, heads, head_dim], heads a multiple of the K/V heads'
        B, p.n, p.H, _ = q.shape
        _rows(cache, q, B, p.n, p.H, 'q')
        _places(p, cache, table, lengths, counts, B)
        p.q_sb, p.q_sn, p.q_sh, _ = q.stride()
        p.scale = scale
        lib = L.load()
        with torch.cuda.device(cache.device):
            if cache.bits == 16 and cache._maps is None:
                maps = C.create_string_buffer(256)
                L.check(lib.ha_paged_maps(C.byref(p), maps), 'ha_paged_maps')
                cache._maps = maps
            p.maps = None if cache._maps is None else C.addressof(cache._maps)
            nbytes = lib.ha_paged_attn_workspace_bytes(C.byref(p))
        L.check(min(nbytes, 0), 'ha_paged_attn')
        return nbytes, _dense(*q.shape), _dense(B, p.H, p.n)

    cache._check_place()
    raw, (nbytes, form, lse_form) = cache._plan(('attn', _form(q), _form(table), _form(lengths), _form(counts), scale), make)
    dev = cache.device
    o = _new(*form, dtype=cache.dtype, device=dev)
    lse = _new(*lse_form, dtype=torch.float32, device=dev)
    p = L.PagedParams.from_buffer_copy(raw)
    ops._set_status(p, dev)
    p.q, p.table, p.lengths, p.o, p.lse = q.data_ptr(), table.data_ptr(), lengths.data_ptr(), o.data_ptr(), lse.data_ptr()
    if nbytes:
        ws = _new((nbytes,), (1,), dtype=torch.uint8, device=dev)        # (free once the launches are enqueued: same stream)
        p.workspace, p.workspace_bytes = ws.data_ptr(), nbytes
    if counts is not None:
        p.counts = counts.data_ptr()
    L.check(ops._call(L.load().ha_paged_attn, dev, C.byref(p)), 'ha_paged_attn')
    return o, lse


def paged_gather(cache, table, lengths, rows):
    """Positions 0 .. rows - 1 of every sequence as dense (k, v) [B, kv_heads, rows, head_dim] in the cache's type, zero from lengths[b] (int32 [B]) on: the
    layout that HyperAttention takes."""
    rows = int(rows)

    def make(p):
        assert table.dim() == 2 and rows >= 0, 'table must be int32 [batch, columns], rows a number'
        _places(p, cache, table, lengths, None, table.shape[0])
        p.rows = rows
        return _dense(table.shape[0], cache.kv_heads, rows, cache.head_dim)

    cache._check_place()
    raw, form = cache._plan(('gather', _form(table), _form(lengths), rows), make)
    p = L.PagedParams.from_buffer_copy(raw)
    ops._set_status(p, cache.device)
    k = _new(*form, dtype=cache.dtype, device=cache.device)
    v = _new(*form, dtype=cache.dtype, device=cache.device)
    p.table, p.lengths, p.k_out, p.v_out = table.data_ptr(), lengths.data_ptr(), k.data_ptr(), v.data_ptr()
    L.check(ops._call(L.load().ha_paged_gather, cache.device, C.byref(p)), 'ha_paged_gather')
    return k, v
