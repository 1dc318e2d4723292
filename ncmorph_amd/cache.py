"""Paged K/V cache on device tensors: what continues a sequence after its
prefill. A step hands over the new rows of some requests (one token each, a
drafted tree of tokens, a chunk of a prompt): `write` puts their K and V into
the cache, `attention` lets their queries read it, `read` gives cached tokens
back as dense rows.

Every call takes the step's requests as three int32 device tensors: offsets
[requests + 1] (request r's rows are offsets[r] .. offsets[r + 1] - 1), starts
[requests] (the tokens of the sequence before them) and page_table [requests,
width] (page_table[r, t // page_size] holds token t). They are read on the
stream, so a captured step follows what they hold at replay; a token past the
table or in a page outside the cache is not there (not written, read as zeros,
not seen), and rows of no request are left as they were. The C ABI's
ncm_kv_cache_t and ncm_kv_batch_t say the rest. The reference has no cache
(its forward, src/decoder.zig:62-228, starts at position 0).
"""
from __future__ import annotations

import ctypes as C

from . import _check as _ck
from ._lib import NCM_E_ARG, NCM_E_SHAPE, NcmError, check, lib
from .context import stream_context

NCM_KV_BF16, NCM_KV_FP8, NCM_KV_INT8 = 0, 1, 2
_CODES = {"bfloat16": NCM_KV_BF16, "float8_e4m3fn": NCM_KV_FP8, "int8": NCM_KV_INT8}


class _Cache(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("k_scale", C.c_void_p),
                ("v_scale", C.c_void_p), ("k_stride", C.c_int64), ("v_stride", C.c_int64),
                ("k_scale_stride", C.c_int64), ("v_scale_stride", C.c_int64),
                ("pages", C.c_int64), ("kv_heads", C.c_int32), ("page_size", C.c_int32),
                ("head_dim", C.c_int32), ("codes", C.c_int32)]


class _Batch(C.Structure):
    _fields_ = [("offsets", C.c_void_p), ("starts", C.c_void_p), ("page_table", C.c_void_p),
                ("requests", C.c_int64), ("rows", C.c_int64), ("table_width", C.c_int64),
                ("table_stride", C.c_int64)]


def _page_stride(t, name, shape, size, where):
    """Elements from a page (of `size`) to the next of a tensor of contiguous
    pages."""
    if t.shape != shape:
        raise NcmError(NCM_E_SHAPE, where, f"{name} has shape {tuple(t.shape)}, expected {shape}")
    if t.is_contiguous():
        return size
    inner, strides = 1, t.stride()
    for d in range(len(shape) - 1, 0, -1):
        if shape[d] != 1 and strides[d] != inner:
            raise NcmError(NCM_E_ARG, where, f"{name} must have contiguous pages")
        inner *= shape[d]
    if shape[0] > 1 and strides[0] < inner:
        raise NcmError(NCM_E_ARG, where, f"{name} must have pages that do not overlap")
    return strides[0] if shape[0] > 1 else inner


class KvCache:
    """One layer's cache: k and v [pages, kv_heads, page_size, head_dim], in
    torch.bfloat16 (as given), torch.float8_e4m3fn or torch.int8 (codes, with
    float32 k_scale and v_scale [pages, kv_heads, page_size]). Pages may lie
    apart, as those of one layer of a buffer [pages, layers, ...] do.
    page_size: a power of two, 16 to 1024; head_dim 64 or 128. It keeps the
    tensors' addresses: where one gets another storage, make a new KvCache."""

    __slots__ = ("k", "v", "k_scale", "v_scale", "struct", "named")

    def __init__(self, k, v, k_scale=None, v_scale=None):
        W = "KvCache"
        pages, heads, page, hd = shape = _ck.dims(k, "k", W, 4)
        name = _ck._dtype(k)
        codes = _CODES.get(name)
        if codes is None:
            raise NcmError(NCM_E_ARG, W, f"k has dtype {name}, expected bfloat16, "
                                         "float8_e4m3fn or int8")
        if getattr(v, "dtype", None) != k.dtype:
            _ck._common(v, "v", W, (name,))
        ks = _page_stride(k, "k", shape, heads * page * hd, W)
        vs = _page_stride(v, "v", shape, heads * page * hd, W)
        if hd not in (64, 128):
            raise NcmError(NCM_E_SHAPE, W, "head_dim must be 64 or 128")
        if not 16 <= page <= 1024 or page & (page - 1):
            raise NcmError(NCM_E_SHAPE, W, "page_size must be a power of two, 16 to 1024")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        if codes == NCM_KV_BF16:
            if k_scale is not None or v_scale is not None:
                raise NcmError(NCM_E_ARG, W, "k_scale and v_scale are for a quantised cache")
            self.named = (k, "k pages"), (v, "v pages")
            self.struct = _Cache(k.data_ptr(), v.data_ptr(), None, None, ks, vs, 0, 0, pages,
                                 heads, page, hd, codes)
            return
        self.named = (k, "k pages"), (v, "v pages"), (k_scale, "k_scale"), (v_scale, "v_scale")
        if k_scale is None or v_scale is None:
            raise NcmError(-1, W, "k_scale and v_scale are required")
        _ck._common(k_scale, "k_scale", W, _ck.F32)
        _ck._common(v_scale, "v_scale", W, _ck.F32)
        kss = _page_stride(k_scale, "k_scale", shape[:3], heads * page, W)
        vss = _page_stride(v_scale, "v_scale", shape[:3], heads * page, W)
        self.struct = _Cache(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
                             ks, vs, kss, vss, pages, heads, page, hd, codes)


def allocate(pages: int, kv_heads: int, page_size: int, head_dim: int, dtype, device) -> KvCache:
    """A KvCache of zeros; dtype as KvCache takes it."""
    import torch

    shape = (pages, kv_heads, page_size, head_dim)
    k, v = (torch.zeros(shape, dtype=dtype, device=device) for _ in range(2))
    if dtype == torch.bfloat16:
        return KvCache(k, v)
    return KvCache(k, v, *(torch.zeros(shape[:3], device=device) for _ in range(2)))


def _batch(a, kv, page_table, offsets, starts, rows):
    """The checked ncm_kv_batch_t of a step."""
    W = a.where
    if not isinstance(kv, KvCache):
        raise NcmError(NCM_E_ARG, W, "kv must be a KvCache")
    (requests,) = _ck.dims(starts, "starts", W, 1)
    _, width = _ck.dims(page_table, "page_table", W, 2)
    ps = a.dev(starts, "starts", _ck.I32, (requests,))
    po = a.dev(offsets, "offsets", _ck.I32, (requests + 1,))
    pt, stride = a.rows(page_table, "page_table", _ck.I32, requests, width)
    a.seen += kv.named
    return _Batch(po, ps, pt, requests, rows, width, max(stride, width))


def _rows(a, t, name, rows, cols):
    """(address, row stride) of bfloat16 rows as the kernels read them."""
    p, stride = a.rows(t, name, _ck.BF16, rows, cols)
    return p, stride if rows > 1 else (cols + 7) // 8 * 8


def write(kv: KvCache, k, v, page_table, offsets, starts, ctx=None):
    """Writes a step's K and V, torch.bfloat16 [rows, >= kv_heads * head_dim]
    with contiguous rows (column slices of a q|k|v buffer are allowed), into
    the cache on torch's current stream, quantised as the cache's dtype says."""
    W = "cache.write"
    a = _ck.Args(W)
    rows, _ = _ck.dims(k, "k", W, 2)
    b = _batch(a, kv, page_table, offsets, starts, rows)
    width = kv.struct.kv_heads * kv.struct.head_dim
    pk, ks = _rows(a, k, "k", rows, width)
    pv, vs = _rows(a, v, "v", rows, width)
    a.done()
    ctx = stream_context(k.device, ctx)
    check(lib().ncm_kv_write_dev(ctx.handle, C.byref(kv.struct), C.byref(b), pk, pv, ks, vs), W)


def read(kv: KvCache, page_table, offsets, starts, rows: int, out=None, ctx=None):
    """(k, v), torch.bfloat16 [rows, kv_heads * head_dim]: what the cache holds
    of the tokens that a write of the same step would write. out: a pair of
    tensors as write takes them, else new ones (whose rows of no request are
    not initialised)."""
    import torch

    W = "cache.read"
    a = _ck.Args(W)
    b = _batch(a, kv, page_table, offsets, starts, rows)
    width = kv.struct.kv_heads * kv.struct.head_dim
    if out is None:
        out = (torch.empty(rows, width, dtype=torch.bfloat16, device=kv.k.device),
               torch.empty(rows, width, dtype=torch.bfloat16, device=kv.k.device))
        pk, pv, ks, vs = out[0].data_ptr(), out[1].data_ptr(), width, width
    else:
        pk, ks = _rows(a, out[0], "out[0]", rows, width)
        pv, vs = _rows(a, out[1], "out[1]", rows, width)
    a.done()
    ctx = stream_context(kv.k.device, ctx)
    check(lib().ncm_kv_read_dev(ctx.handle, C.byref(kv.struct), C.byref(b), pk, pv, ks, vs), W)
    return out[0], out[1]


def attention(q, kv: KvCache, q_heads: int, page_table, offsets, starts, tree_mask=None,
              window: int = 0, positions=None, scale: float | None = None, out=None,
              workspace=None, ctx=None):
    """Attention of a step's queries, torch.bfloat16 [rows, >= q_heads *
    head_dim] with contiguous rows, over the cache, which holds the step's own
    K and V already; torch.bfloat16 [rows, q_heads * head_dim]. A row sees the
    tokens before its request's rows and of those rows the ones whose bit its
    tree_mask sets: int64 or uint64 [rows, words], bit j % 64 of word j // 64
    for its request's row j; without a tree_mask its own and the earlier ones.
    window > 0: of the tokens before (without a tree_mask, of all tokens) those
    less than window positions back from the row's position, positions[row]
    (int32) or starts + its index. Rows that see nothing get zeros.
    scale: head_dim ** -0.5 by default. out may be q; a new one's rows of no
    request are not initialised. workspace: uint8 scratch, taken from torch's
    allocator where not given."""
    import torch

    W = "cache.attention"
    a = _ck.Args(W)
    rows, _ = _ck.dims(q, "q", W, 2)
    b = _batch(a, kv, page_table, offsets, starts, rows)
    hd = kv.struct.head_dim
    pq, qs = _rows(a, q, "q", rows, q_heads * hd)
    words = 0
    if tree_mask is not None:
        _, words = _ck.dims(tree_mask, "tree_mask", W, 2)
    pm = a.dev(tree_mask, "tree_mask", _ck.U64, (rows, words), optional=True)
    if tree_mask is not None and words == 0:
        pm = b.offsets  # a mask of no words has no address of its own; nothing is read there
    pp = a.dev(positions, "positions", _ck.I32, (rows,), optional=True)
    need = C.c_size_t()
    check(lib().ncm_kv_attention_workspace(C.byref(kv.struct), C.byref(b), q_heads,
                                           C.byref(need)), W)
    if out is None:
        out = torch.empty(rows, q_heads * hd, dtype=torch.bfloat16, device=q.device)
        po, os_ = out.data_ptr(), q_heads * hd
    else:
        po, os_ = _rows(a, out, "out", rows, q_heads * hd)
    if workspace is None:
        workspace = torch.empty(need.value, dtype=torch.uint8, device=q.device)
        pw = workspace.data_ptr()
    else:
        pw = a.dev(workspace, "workspace", ("uint8",))
    a.done()
    ctx = stream_context(q.device, ctx)
    check(lib().ncm_kv_attention_dev(ctx.handle, C.byref(kv.struct), C.byref(b), pq, po, q_heads,
                                     qs, os_, hd ** -0.5 if scale is None else scale, window, pp,
                                     pm, words, pw,
                                     workspace.numel()), W)
    return out
