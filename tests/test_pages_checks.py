"""Refusals of the page pool's calls, on the CPU: the wrappers' and the C ABI's,
and the layout of its struct."""
import ctypes as C
import os
import subprocess

import pytest
import torch

from ncmorph_amd import cache
from ncmorph_amd._lib import NCM_E_ARG, NCM_E_NULL, NCM_E_SHAPE, NcmError, lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
i32 = torch.int32


def _raises(status, fn, *a, **kw):
    with pytest.raises(NcmError) as e:
        fn(*a, **kw)
    assert e.value.status == status, str(e.value)
    return str(e.value)


def z(*shape, dtype=i32):
    return torch.zeros(shape, dtype=dtype)


def test_wrappers():
    P = cache.PagePool
    pool = P(z(8), z(1), z(8))
    _raises(NCM_E_SHAPE, P, z(8), z(2), z(8))
    _raises(NCM_E_SHAPE, P, z(8), z(1), z(7))
    _raises(NCM_E_SHAPE, P, z(0), z(1), z(0))
    _raises(NCM_E_SHAPE, P, z(2, 4), z(1), z(8))
    _raises(NCM_E_ARG, P, z(8).long(), z(1), z(8))
    _raises(NCM_E_ARG, P, z(16)[::2], z(1), z(8))
    t, l = z(3, 5), z(3)
    E = cache.extend
    assert "GPU" in _raises(NCM_E_ARG, E, pool, t, l, l, 4, 16)
    _raises(NCM_E_ARG, E, (z(8),), t, l, l, 4, 16)
    _raises(NCM_E_SHAPE, E, pool, t, z(4), l, 4, 16)
    _raises(NCM_E_ARG, E, pool, t, l.long(), l, 4, 16)
    _raises(NCM_E_NULL, E, pool, t, l, None, 4, 16)
    _raises(NCM_E_ARG, E, pool, z(5, 3).t(), l, l, 4, 16)
    _raises(NCM_E_SHAPE, E, pool, t, l, l, 4, 16, tree_mask=z(3, 1, dtype=torch.int64))
    _raises(NCM_E_ARG, E, pool, t, l, l, 4, 16, tree_mask=z(4, 1))
    _raises(NCM_E_SHAPE, E, pool, t, l, l, -1, 16)
    for fn in (cache.share, cache.release):
        assert "GPU" in _raises(NCM_E_ARG, fn, pool, t, l, l, 16)
        _raises(NCM_E_ARG, fn, None, t, l, l, 16)
        _raises(NCM_E_SHAPE, fn, pool, t, l, z(2), 16)
        _raises(NCM_E_SHAPE, fn, pool, z(3), l, l, 16)


def test_library(ncm):
    L, p, no = lib(), 1 << 20, None
    ctx = C.c_void_p(p)

    def pool(**k):
        return C.byref(cache._Pool(**dict(dict(free=p, count=p, refs=p, marks=p, pages=8), **k)))

    def E(**k):
        d = dict(ctx=ctx, pool=pool(), added=p, starts=p, table=p, requests=2, width=4, stride=4,
                 page=16, rows=3, mask=no, words=0, offsets=p, positions=p, slots=p, missing=p,
                 space=p)
        return L.ncm_pages_extend_dev(*dict(d, **k).values())

    for bad in (dict(requests=-1), dict(requests=1 << 16), dict(width=-1), dict(stride=3),
                dict(page=8), dict(page=24), dict(page=2048), dict(rows=-1),
                dict(rows=(1 << 30) + 1), dict(width=1 << 27, stride=1 << 27), dict(words=-1),
                dict(pool=pool(pages=0)), dict(pool=pool(pages=(1 << 30) + 1))):
        assert E(**bad) == NCM_E_SHAPE, bad
    for bad in (dict(ctx=no), dict(added=no), dict(starts=no), dict(table=no), dict(offsets=no),
                dict(positions=no), dict(slots=no), dict(missing=no), dict(space=no),
                dict(pool=pool(free=no)), dict(pool=pool(marks=no))):
        assert E(**bad) == NCM_E_NULL, bad
    for bad in (dict(slots=p + 4), dict(mask=p + 4, words=1), dict(pool=pool(marks=p + 4))):
        assert E(**bad) == NCM_E_ARG, bad

    def two(fn, tail):
        def call(**k):
            d = dict(ctx=ctx, pool=pool(), table=p, a=p, b=p, requests=2, width=4, stride=4,
                     page=16)
            return fn(*dict(d, **k).values(), *tail)
        return call

    for call in (two(L.ncm_pages_share_dev, ()), two(L.ncm_pages_release_dev, (p,))):
        for bad in (dict(ctx=no), dict(pool=no), dict(a=no), dict(b=no), dict(table=no)):
            assert call(**bad) == NCM_E_NULL, bad
        for bad in (dict(requests=1 << 16), dict(stride=3), dict(page=0)):
            assert call(**bad) == NCM_E_SHAPE, bad
        assert call(requests=0) == 0 and call(width=0) == 0
    assert two(L.ncm_pages_release_dev, (no,))() == NCM_E_NULL


def test_layout(tmp_path):
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "ncmorph_amd.h"',
             "int main(void) {", 'printf("%zu\\n", sizeof(ncm_page_pool_t));']
    lines += [f'printf("%zu\\n", offsetof(ncm_page_pool_t, {f}));' for f, _ in cache._Pool._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0;", "}"]))
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o",
                    str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout
    assert [int(x) for x in out.split()] == [C.sizeof(cache._Pool)] + [
        getattr(cache._Pool, f).offset for f, _ in cache._Pool._fields_]
