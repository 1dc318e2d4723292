"""Refusals of the 4-bit products, on the CPU: the wrappers' and the C ABI's,
and the layout of the weight's struct."""
import ctypes as C
import os
import subprocess

import pytest
import torch

from ncmorph_amd import kernels
from ncmorph_amd._lib import NCM_E_ARG, NCM_E_LENGTH, NCM_E_NULL, NCM_E_SHAPE, NcmError, lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
bf, u8 = torch.bfloat16, torch.uint8


def _raises(status, fn, *a, **kw):
    with pytest.raises(NcmError) as e:
        fn(*a, **kw)
    assert e.value.status == status, str(e.value)
    return str(e.value)


def z(*shape, dtype=bf):
    return torch.zeros(shape, dtype=dtype)


def test_wrappers(ncm):
    P, Q, K = kernels.pack_int4, kernels.quantise_int4, kernels.linear_int4
    codes, scales = z(20, 136, dtype=u8), z(20, 3)
    assert "GPU" in _raises(NCM_E_ARG, P, codes, scales, 64)
    _raises(NCM_E_SHAPE, P, codes, scales, 128)
    _raises(NCM_E_SHAPE, P, codes, scales, 16)
    _raises(NCM_E_SHAPE, P, codes, scales, 256)
    _raises(NCM_E_SHAPE, P, z(20, 132, dtype=u8), scales, 64)
    _raises(NCM_E_SHAPE, P, z(20, 0, dtype=u8), z(20, 0), 64)
    _raises(NCM_E_ARG, P, codes.int(), scales, 64)
    _raises(NCM_E_ARG, P, codes, scales.float(), 64)
    _raises(NCM_E_SHAPE, P, codes, scales, 64, zeros=z(20, 2, dtype=u8))
    _raises(NCM_E_ARG, P, codes, scales, 64, zeros=z(20, 3))
    _raises(NCM_E_ARG, P, z(136, 20, dtype=u8).t(), scales, 64)
    assert "GPU" in _raises(NCM_E_ARG, Q, z(20, 136), 64)
    _raises(NCM_E_ARG, Q, z(20, 136).float(), 64)
    _raises(NCM_E_SHAPE, Q, z(20, 130), 64)
    _raises(NCM_E_ARG, Q, z(136, 24).t(), 64)
    W = kernels.Int4Weight
    pc, ps = z(2 * 2 * 1024, dtype=u8), z(2 * 2 * 2 * 32, dtype=u8)
    w = W(pc, ps, 20, 136, 64, False)
    _raises(NCM_E_SHAPE, W, pc, ps, 20, 136, 64, True)
    _raises(NCM_E_SHAPE, W, pc, ps, 33, 136, 64, False)
    _raises(NCM_E_ARG, W, pc.view(torch.int8), ps, 20, 136, 64, False)
    x = z(3, 136)
    assert "GPU" in _raises(NCM_E_ARG, K, x, w)
    _raises(NCM_E_ARG, K, x, codes)
    _raises(NCM_E_SHAPE, K, z(3, 128), w)
    _raises(NCM_E_ARG, K, x.float(), w)
    _raises(NCM_E_ARG, K, z(136, 3).t(), w)
    _raises(NCM_E_SHAPE, K, x, w, bias=z(19))
    _raises(NCM_E_ARG, K, x, w, residual=z(3, 20))
    _raises(NCM_E_SHAPE, K, x, w, residual=z(3, 21, dtype=torch.float32))
    _raises(NCM_E_ARG, K, x, w, out_mode="fp8")
    _raises(NCM_E_ARG, K, x, w, out=z(3, 20))
    _raises(NCM_E_SHAPE, K, x, w, out=z(2, 20), out_mode="bf16")
    _raises(NCM_E_ARG, K, x, w, workspace=z(64))


def test_library(ncm):
    L, p, no = lib(), 1 << 20, None
    ctx = C.c_void_p(p)

    def weight(**k):
        return C.byref(kernels._Int4(**dict(dict(codes=p, scales=p, n=20, k=136, group=64,
                                                 has_zeros=0), **k)))

    def Y(**k):
        d = dict(ctx=ctx, x=p, stride=136, w=weight(), bias=no, residual=no, y=p, m=3, mode=0,
                 ws=no, size=0)
        return L.ncm_linear_int4(*dict(d, **k).values())

    for bad in (dict(ctx=no), dict(w=no), dict(x=no), dict(y=no), dict(w=weight(codes=no)),
                dict(w=weight(scales=no))):
        assert Y(**bad) == NCM_E_NULL, bad
    for bad in (dict(m=-1), dict(m=(1 << 20) + 1), dict(stride=128), dict(w=weight(k=132)),
                dict(w=weight(k=0)), dict(w=weight(n=-1)), dict(w=weight(group=48)),
                dict(w=weight(n=1 << 28, k=1 << 10)), dict(w=weight(n=(1 << 26) + 1, k=8),
                                                           stride=8)):
        assert Y(**bad) == NCM_E_SHAPE, bad
    for bad in (dict(mode=3), dict(x=p + 8), dict(stride=140), dict(y=p + 2), dict(bias=p + 1),
                dict(residual=p + 2), dict(w=weight(codes=p + 8)), dict(w=weight(scales=p + 8)),
                dict(residual=p, y=p, mode=2)):
        assert Y(**bad) == NCM_E_ARG, bad
    big = weight(n=256, k=4096)
    assert Y(w=big, stride=4096, m=64) == NCM_E_NULL
    assert Y(w=big, stride=4096, m=64, ws=p) == NCM_E_LENGTH
    assert Y(w=big, stride=4096, m=64, ws=p + 4, size=1 << 30) == NCM_E_ARG
    need = C.c_size_t()
    ws = L.ncm_linear_int4_workspace
    assert ws(64, 256, 4096, C.byref(need)) == 0 and need.value % (64 * 256 * 4) == 0 < need.value
    assert ws(16, 256, 4096, C.byref(need)) == 0 and need.value == 0
    assert ws(16, 256, 4096, None) == NCM_E_NULL and ws(-1, 256, 4096, C.byref(need)) == NCM_E_SHAPE
    assert Y(m=0) == 0 and Y(w=weight(n=0)) == 0
    a, b = C.c_size_t(), C.c_size_t()
    assert L.ncm_int4_bytes(20, 136, 64, 0, C.byref(a), C.byref(b)) == 0
    assert (a.value, b.value) == (4096, 256)
    assert L.ncm_int4_bytes(20, 136, 32, 1, C.byref(a), C.byref(b)) == 0 and b.value == 1024
    assert L.ncm_int4_bytes(20, 136, 64, 0, None, C.byref(b)) == NCM_E_NULL
    pack = lambda **k: L.ncm_int4_pack_dev(*dict(dict(  # noqa: E731
        ctx=ctx, codes=p, scales=p, zeros=no, n=20, k=136, group=64, to=p, sto=p), **k).values())
    assert pack(ctx=no) == NCM_E_NULL and pack(codes=no) == NCM_E_NULL and pack(to=no) == NCM_E_NULL
    assert pack(k=4) == NCM_E_SHAPE and pack(to=p + 4) == NCM_E_ARG and pack(n=0) == 0
    quant = lambda **k: L.ncm_int4_quantise_dev(*dict(dict(  # noqa: E731
        ctx=ctx, w=p, n=20, k=136, stride=136, group=64, codes=p, scales=p, zeros=no), **k).values())
    assert quant(ctx=no) == NCM_E_NULL and quant(w=no) == NCM_E_NULL
    assert quant(stride=135) == NCM_E_SHAPE and quant(group=0) == NCM_E_SHAPE and quant(n=0) == 0


def test_layout(tmp_path):
    fields = kernels._Int4._fields_
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "ncmorph_amd.h"',
             "int main(void) {", 'printf("%zu\\n", sizeof(ncm_int4_weight_t));']
    lines += [f'printf("%zu\\n", offsetof(ncm_int4_weight_t, {f}));' for f, _ in fields]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0;", "}"]))
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o",
                    str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout
    assert [int(x) for x in out.split()] == [C.sizeof(kernels._Int4)] + [
        getattr(kernels._Int4, f).offset for f, _ in fields]
