"""Refusals of cache.attention with groups, on the CPU."""
import ctypes as C

import pytest
import torch

from ncmorph_amd import cache
from ncmorph_amd._lib import NCM_E_ARG, NCM_E_LENGTH, NCM_E_NULL, NCM_E_SHAPE, NcmError, lib

bf, i32 = torch.bfloat16, torch.int32


def z(*shape, dtype=i32):
    return torch.zeros(shape, dtype=dtype)


def _raises(status, *a, **kw):
    with pytest.raises(NcmError) as e:
        cache.attention(*a, **kw)
    assert e.value.status == status, str(e.value)
    return str(e.value)


def test_wrapper(ncm):
    kv = cache.KvCache(z(4, 2, 16, 64, dtype=bf), z(4, 2, 16, 64, dtype=bf))
    args = (z(3, 256, dtype=bf), kv, 4, z(3, 5), z(4), z(3))
    good = dict(groups=z(3), shared=z(2))
    assert "GPU" in _raises(NCM_E_ARG, *args, **good)
    _raises(NCM_E_NULL, *args, groups=z(3))
    _raises(NCM_E_NULL, *args, shared=z(3))
    _raises(NCM_E_SHAPE, *args, groups=z(2), shared=z(2))
    _raises(NCM_E_SHAPE, *args, groups=z(5), shared=z(4))      # more groups than requests
    _raises(NCM_E_ARG, *args, groups=z(3).long(), shared=z(2))
    _raises(NCM_E_ARG, *args, groups=z(3), shared=z(2, dtype=torch.float32))
    _raises(NCM_E_ARG, *args, groups=z(6)[::2], shared=z(2))


def test_library(ncm):
    L, p, no = lib(), 1 << 20, None

    def kv(**k):
        d = dict(k=p, v=p, k_scale=no, v_scale=no, k_stride=2048, v_stride=2048,
                 k_scale_stride=0, v_scale_stride=0, pages=1, kv_heads=2, page_size=16,
                 head_dim=64, codes=0)
        return C.byref(cache._Cache(**dict(d, **k)))

    def batch(**k):
        d = dict(offsets=p, starts=p, page_table=p, requests=2, rows=2, table_width=1,
                 table_stride=1)
        return C.byref(cache._Batch(**dict(d, **k)))

    def A(**k):
        d = dict(ctx=C.c_void_p(p), kv=kv(), b=batch(), groups=p, shared=p, n=1, q=p, out=p,
                 heads=4, qs=256, os=256, scale=1.0, window=0, positions=no, mask=no, words=0,
                 ws=p, size=1 << 40)
        return L.ncm_kv_attention_shared_dev(*dict(d, **k).values())

    for bad in (dict(ctx=no), dict(kv=no), dict(b=no), dict(groups=no), dict(shared=no),
                dict(q=no), dict(out=no), dict(ws=no)):
        assert A(**bad) == NCM_E_NULL, bad
    for bad in (dict(n=-1), dict(n=3), dict(heads=3), dict(heads=0), dict(qs=255), dict(window=-1),
                dict(words=-1), dict(kv=kv(head_dim=32)), dict(b=batch(rows=-1)),
                dict(b=batch(rows=1 << 30), heads=64, qs=4096, os=4096)):
        assert A(**bad) == NCM_E_SHAPE, bad
    assert A(ws=p + 8) == NCM_E_ARG and A(q=p + 2) == NCM_E_ARG
    assert A(b=batch(rows=0)) == 0 and A(b=batch(requests=0), n=0) == 0
    size = C.c_size_t(7)
    W = L.ncm_kv_attention_shared_workspace
    assert W(kv(), batch(), 1, 4, None) == NCM_E_NULL
    assert W(kv(), batch(), 3, 4, C.byref(size)) == NCM_E_SHAPE and size.value == 0
    assert W(kv(), batch(), 1, 4, C.byref(size)) == 0 and size.value > 0
    assert A(size=size.value - 1) == NCM_E_LENGTH
