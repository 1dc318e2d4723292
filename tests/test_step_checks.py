"""Argument checks of the operators that continue a sequence, on the CPU: every
tensor's dtype and shape before any call, the C ABI's refusals, and the layouts
of its structs."""
import ctypes as C
import os
import subprocess

import pytest
import torch

from ncmorph_amd import cache, kernels
from ncmorph_amd._lib import NCM_E_ARG, NCM_E_NULL, NCM_E_SHAPE, NcmError, lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
bf, f32, i32, i64, i8 = torch.bfloat16, torch.float32, torch.int32, torch.int64, torch.int8


def _raises(status, fn, *a, **kw):
    with pytest.raises(NcmError) as e:
        fn(*a, **kw)
    assert e.value.status == status, str(e.value)
    return str(e.value)


def z(*shape, dtype=bf):
    return torch.zeros(shape, dtype=dtype)


def test_cache_checks():
    K = cache.KvCache
    p = z(4, 2, 16, 64)
    K(p, z(4, 2, 16, 64))
    _raises(NCM_E_SHAPE, K, p, z(4, 2, 16, 128))
    _raises(NCM_E_SHAPE, K, z(4, 2, 16, 96), z(4, 2, 16, 96))
    for page in (8, 24, 2048):
        _raises(NCM_E_SHAPE, K, z(4, 2, page, 64), z(4, 2, page, 64))
    _raises(NCM_E_SHAPE, K, z(4, 2, 16), z(4, 2, 16))
    _raises(NCM_E_ARG, K, p.float(), p.float())
    _raises(NCM_E_ARG, K, p, z(4, 2, 16, 64, dtype=i8))
    _raises(NCM_E_ARG, K, p, p, z(4, 2, 16, dtype=f32), z(4, 2, 16, dtype=f32))
    q, s = z(4, 2, 16, 64, dtype=i8), z(4, 2, 16, dtype=f32)
    K(q, q, s, s)
    _raises(NCM_E_NULL, K, q, q)
    _raises(NCM_E_NULL, K, q, q, s, None)
    _raises(NCM_E_SHAPE, K, q, q, s, z(4, 2, 17, dtype=f32))
    _raises(NCM_E_ARG, K, q, q, s, z(4, 2, 16))
    _raises(NCM_E_ARG, K, z(4, 2, 64, 16).transpose(2, 3), p)      # inside a page
    _raises(NCM_E_ARG, K, z(1, 2, 16, 64).expand(4, 2, 16, 64), p)  # pages that overlap
    both = z(4, 2, 2, 16, 64)
    assert K(both[:, 0], both[:, 1]).struct.k_stride == 2 * 2 * 16 * 64


def test_step_tensors():
    kv = cache.KvCache(z(4, 2, 16, 64), z(4, 2, 16, 64))
    x, t, o, s = z(3, 128), z(2, 5, dtype=i32), z(3, dtype=i32), z(2, dtype=i32)
    w = cache.write
    assert "GPU" in _raises(NCM_E_ARG, w, kv, x, x, t, o, s)
    _raises(NCM_E_ARG, w, (x, x), x, x, t, o, s)
    _raises(NCM_E_SHAPE, w, kv, x, z(2, 128), t, o, s)
    _raises(NCM_E_SHAPE, w, kv, z(3, 64), x, t, o, s)
    _raises(NCM_E_ARG, w, kv, x.float(), x, t, o, s)
    _raises(NCM_E_SHAPE, w, kv, x, x, t, z(2, dtype=i32), s)
    _raises(NCM_E_SHAPE, w, kv, x, x, z(3, 5, dtype=i32), o, s)
    _raises(NCM_E_ARG, w, kv, x, x, t, o.long(), s)
    _raises(NCM_E_ARG, w, kv, x, x, t.long(), o, s)
    _raises(NCM_E_ARG, w, kv, x, x, z(5, 2, dtype=i32).t(), o, s)
    _raises(NCM_E_SHAPE, cache.read, kv, t, o, s, 3, out=(x, z(4, 128)))
    _raises(NCM_E_ARG, cache.read, kv, t, o, s, 3, out=(x, x.float()))
    q, att = z(3, 256), cache.attention
    assert "GPU" in _raises(NCM_E_ARG, att, q, kv, 4, t, o, s)
    _raises(NCM_E_SHAPE, att, z(3, 192), kv, 4, t, o, s)
    _raises(NCM_E_SHAPE, att, q, kv, 4, t, o, s, tree_mask=z(2, 1, dtype=i64))
    _raises(NCM_E_ARG, att, q, kv, 4, t, o, s, tree_mask=z(3, 1, dtype=i32))
    _raises(NCM_E_SHAPE, att, q, kv, 4, t, o, s, positions=z(4, dtype=i32))
    _raises(NCM_E_SHAPE, att, q, kv, 4, t, o, s, out=z(3, 255))
    _raises(NCM_E_ARG, att, q, kv, 4, t, o, s, out=z(3, 256, dtype=f32))
    _raises(NCM_E_ARG, att, q, kv, 4, t, o, s, workspace=z(8, dtype=f32))
    _raises(NCM_E_SHAPE, att, z(3, 192), kv, 3, t, o, s)             # 3 heads over 2


def test_context_of_another_device():
    from types import SimpleNamespace

    from ncmorph_amd.context import stream_context

    _raises(NCM_E_ARG, stream_context, torch.device("cuda", 0), SimpleNamespace(device=1))


def test_rope_and_logits_checks():
    x, p, f = z(5, 128), z(5, dtype=i32), z(32, dtype=f32)
    r = kernels.rope_positions
    assert "GPU" in _raises(NCM_E_ARG, r, x, p, f, 2, 64)
    _raises(NCM_E_SHAPE, r, x, p, f, 3, 64)
    _raises(NCM_E_SHAPE, r, x, z(4, dtype=i32), f, 2, 64)
    _raises(NCM_E_ARG, r, x, p.long(), f, 2, 64)
    _raises(NCM_E_ARG, r, x.half(), p, f, 2, 64)
    _raises(NCM_E_ARG, r, x, p, f, 2, 64, layout="both")
    _raises(NCM_E_ARG, r, x, p, f, 2, 64, out=z(5, 128, dtype=f32))
    _raises(NCM_E_SHAPE, r, x, p, f, 2, 64, out=z(5, 127))
    a, l = kernels.adjust_logits, z(2, 50, dtype=f32)
    assert "GPU" in _raises(NCM_E_ARG, a, l)
    _raises(NCM_E_SHAPE, a, l, history=z(3, 4, dtype=i32))
    _raises(NCM_E_NULL, a, l, prompt_lens=z(2, dtype=i32))
    _raises(NCM_E_NULL, a, l, bias_ids=z(2, 3, dtype=i32))
    _raises(NCM_E_NULL, a, l, draft_tokens=z(2, dtype=i32))
    _raises(NCM_E_NULL, a, l, tree_mask=z(2, 1, dtype=i64))
    _raises(NCM_E_SHAPE, a, l, allowed=z(2, 1, dtype=i32))
    _raises(NCM_E_SHAPE, a, l, offsets=z(0, dtype=i32))
    _raises(NCM_E_ARG, a, l, repetition=z(2, dtype=torch.float64))


def test_library_refuses(ncm):
    """The C ABI's own checks, before any device work: a context handle is
    only looked at after them."""
    L, no = lib(), None
    buf = (C.c_char * 64)()
    p = C.addressof(buf) + (-C.addressof(buf)) % 16
    ctx = C.c_void_p(p)
    R = lambda **k: L.ncm_rope_positions_dev(*[dict(  # noqa: E731
        ctx=ctx, x=p, y=p, pos=p, inv=p, rows=1, heads=2, hd=64, rot=64, xs=128, ys=128, lay=0,
        scale=1.0, dt=0, **{})[n] if n not in k else k[n] for n in
        ("ctx", "x", "y", "pos", "inv", "rows", "heads", "hd", "rot", "xs", "ys", "lay", "scale",
         "dt")])
    assert R(ctx=no) == NCM_E_NULL and R(x=no) == NCM_E_NULL and R(inv=no) == NCM_E_NULL
    for bad in (dict(rows=-1), dict(rows=1 << 31), dict(rows=(1 << 25) + 1), dict(rot=63), dict(rot=66), dict(rot=0),
                dict(xs=127), dict(ys=127), dict(heads=-1), dict(hd=0)):
        assert R(**bad) == NCM_E_SHAPE, bad
    for bad in (dict(lay=2), dict(dt=1), dict(ys=130)):
        assert R(**bad) == NCM_E_ARG, bad
    assert R(rows=0) == 0 and R(heads=0) == 0

    def kv(**k):
        d = dict(k=p, v=p, k_scale=no, v_scale=no, k_stride=2048, v_stride=2048,
                 k_scale_stride=0, v_scale_stride=0, pages=1, kv_heads=2, page_size=16,
                 head_dim=64, codes=0)
        return C.byref(cache._Cache(**dict(d, **k)))

    def batch(**k):
        d = dict(offsets=p, starts=p, page_table=p, requests=1, rows=1, table_width=1,
                 table_stride=1)
        return C.byref(cache._Batch(**dict(d, **k)))

    W = lambda c, b, k=p, v=p, ks=128, vs=128: L.ncm_kv_write_dev(ctx, c, b, k, v, ks, vs)  # noqa
    assert W(no, batch()) == NCM_E_NULL and W(kv(), no) == NCM_E_NULL
    assert L.ncm_kv_write_dev(no, kv(), batch(), p, p, 128, 128) == NCM_E_NULL
    for bad in (dict(page_size=0), dict(page_size=17), dict(head_dim=32), dict(k_stride=2047),
                dict(pages=0), dict(pages=1 << 31), dict(kv_heads=0)):
        assert W(kv(**bad), batch()) == NCM_E_SHAPE, bad
    s = dict(codes=2, k_scale=p, v_scale=p, k_scale_stride=32, v_scale_stride=32)
    for bad in (dict(codes=3), dict(k=p + 8), dict(k_stride=2049), dict(s, k_scale=p + 4),
                dict(s, v_scale_stride=33)):
        assert W(kv(**bad), batch()) == NCM_E_ARG, bad
    for bad in (dict(k=no), dict(codes=1), dict(k_scale=p), dict(s, v_scale=no)):
        assert W(kv(**bad), batch()) == NCM_E_NULL, bad
    assert W(kv(**dict(s, k_scale_stride=31)), batch()) == NCM_E_SHAPE
    for bad in (dict(requests=-1), dict(requests=1 << 20), dict(rows=1 << 31),
                dict(table_width=2), dict(table_width=-1)):
        assert W(kv(), batch(**bad)) == NCM_E_SHAPE, bad
    for bad in (dict(offsets=no), dict(starts=no), dict(page_table=no)):
        assert W(kv(), batch(**bad)) == NCM_E_NULL, bad
    assert W(kv(), batch(), ks=127) == NCM_E_SHAPE and W(kv(), batch(), ks=132) == NCM_E_ARG
    assert W(kv(), batch(), k=p + 8) == NCM_E_ARG and W(kv(), batch(), v=no) == NCM_E_NULL
    assert L.ncm_kv_read_dev(ctx, kv(), batch(), p, p, 128, 127) == NCM_E_SHAPE
    assert W(kv(), batch(rows=0)) == 0 and W(kv(), batch(requests=0)) == 0

    A = lambda c=None, b=None, q=p, o=p, h=4, qs=256, os_=256, win=0, m=no, mw=0, w=p, n=1 << 40: (  # noqa
        L.ncm_kv_attention_dev(ctx, c or kv(), b or batch(), q, o, h, qs, os_, 1.0, win, no, m, mw,
                               w, n))
    assert A(h=3) == NCM_E_SHAPE and A(h=0) == NCM_E_SHAPE and A(qs=255) == NCM_E_SHAPE
    assert A(win=-1) == NCM_E_SHAPE and A(mw=-1) == NCM_E_SHAPE and A(os_=260) == NCM_E_ARG
    assert A(q=no) == NCM_E_NULL and A(o=p + 2) == NCM_E_ARG
    assert A(b=batch(rows=0)) == 0
    size = C.c_size_t(7)
    assert L.ncm_kv_attention_workspace(kv(), batch(), 4, None) == NCM_E_NULL
    assert L.ncm_kv_attention_workspace(kv(head_dim=1), batch(), 4, C.byref(size)) == NCM_E_SHAPE
    assert L.ncm_kv_attention_workspace(kv(), batch(), 4, C.byref(size)) == 0

    def rules(**k):
        return C.byref(kernels._LogitRules(**dict(dict(requests=2), **k)))

    J = lambda r, x=p, y=p, rows=2, v=50, a=50, b=50, dt=0: L.ncm_adjust_logits_dev(  # noqa: E731
        ctx, r, x, y, rows, v, a, b, dt)
    assert J(no) == NCM_E_NULL and J(rules(), x=no) == NCM_E_NULL
    for r in (rules(draft_tokens=p), rules(bias_ids=p), rules(bias_values=p)):
        assert J(r) == NCM_E_NULL
    assert J(rules(requests=3)) == NCM_E_SHAPE and J(rules(), a=49) == NCM_E_SHAPE
    assert J(rules(offsets=p, requests=1 << 20)) == NCM_E_SHAPE
    assert J(rules(history_width=-1)) == NCM_E_SHAPE and J(rules(), v=-1) == NCM_E_SHAPE
    assert J(rules(), dt=1) == NCM_E_ARG and J(rules(), b=51) == NCM_E_ARG
    assert J(rules(), x=p + 2) == NCM_E_ARG
    assert J(rules(requests=0), rows=0) == 0 and J(rules(), v=0) == 0


def test_struct_layouts_match_header(tmp_path):
    structs = {"ncm_kv_cache_t": cache._Cache, "ncm_kv_batch_t": cache._Batch,
               "ncm_logit_rules_t": kernels._LogitRules}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "ncmorph_amd.h"',
             "int main(void) {"]
    for name, cls in structs.items():
        lines.append(f'printf("{name} size %zu\\n", sizeof({name}));')
        lines += [f'printf("{name} {f} %zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0;", "}"]))
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o",
                    str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout
    got = {tuple(l.split()[:2]): int(l.split()[2]) for l in out.splitlines()}
    for name, cls in structs.items():
        assert C.sizeof(cls) == got[(name, "size")]
        for f, _ in cls._fields_:
            assert getattr(cls, f).offset == got[(name, f)], (name, f)
