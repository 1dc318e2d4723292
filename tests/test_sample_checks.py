"""Refusals of kernels.sample, on the CPU: the wrapper's and the C ABI's, and
the layout of its struct."""
import ctypes as C
import os
import subprocess

import pytest
import torch

from ncmorph_amd import kernels
from ncmorph_amd._lib import NCM_E_ARG, NCM_E_LENGTH, NCM_E_NULL, NCM_E_SHAPE, NcmError, lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _raises(status, *a, **kw):
    with pytest.raises(NcmError) as e:
        kernels.sample(*a, **kw)
    assert e.value.status == status, str(e.value)
    return str(e.value)


def z(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


def test_wrapper(ncm):
    x, u, i32 = z(3, 50), z(3), torch.int32
    assert "GPU" in _raises(NCM_E_ARG, x, u)
    _raises(NCM_E_ARG, x.half(), u)
    _raises(NCM_E_SHAPE, z(50), u)
    _raises(NCM_E_ARG, z(50, 3).t(), u)
    _raises(NCM_E_SHAPE, x, z(2))
    _raises(NCM_E_ARG, x, u.half())
    _raises(NCM_E_NULL, x, None)
    for name, good in (("temperature", torch.float32), ("top_k", i32), ("top_p", torch.float32),
                       ("min_p", torch.float32)):
        _raises(NCM_E_SHAPE, x, u, **{name: z(2, dtype=good)})
        _raises(NCM_E_ARG, x, u, **{name: z(3, dtype=torch.float64)})
        _raises(NCM_E_SHAPE, x, u, offsets=z(3, dtype=i32), **{name: z(3, dtype=good)})
    _raises(NCM_E_SHAPE, x, u, offsets=z(0, dtype=i32))
    _raises(NCM_E_SHAPE, x, u, out=z(4, dtype=i32))
    _raises(NCM_E_ARG, x, u, out=z(3))
    _raises(NCM_E_ARG, x, u, workspace=z(3))
    _raises(NCM_E_SHAPE, z(1, (1 << 20) + 1), z(1))


def test_library(ncm):
    L, p, no = lib(), 1 << 20, None

    def S(**k):
        d = dict(ctx=C.c_void_p(p), rules=None, x=p, rows=2, vocab=50, stride=50, dtype=0, u=p,
                 bits=32, tokens=p, chance=no, ws=p, size=1 << 40)
        r = {n: k.pop(n) for n in [f for f, _ in kernels._SampleRules._fields_] if n in k}
        d["rules"] = C.byref(kernels._SampleRules(**dict(dict(requests=2), **r)))
        return L.ncm_sample_dev(*dict(d, **k).values())

    for bad in (dict(rows=-1), dict(rows=1 << 22), dict(vocab=-1), dict(vocab=(1 << 20) + 1),
                dict(stride=49), dict(requests=3), dict(requests=-1),
                dict(offsets=p, requests=1 << 16)):
        assert S(**bad) == NCM_E_SHAPE, bad
    for bad in (dict(ctx=no), dict(rules=no), dict(x=no), dict(u=no), dict(tokens=no)):
        assert S(**bad) == NCM_E_NULL, bad
    for bad in (dict(dtype=1), dict(bits=16), dict(x=p + 2), dict(u=p + 2), dict(u=p + 4, bits=64)):
        assert S(**bad) == NCM_E_ARG, bad
    assert S(rows=0, requests=0) == 0 and S(offsets=p, requests=0) == 0
    size = C.c_size_t()
    assert L.ncm_sample_workspace(2, 50, None) == NCM_E_NULL
    assert L.ncm_sample_workspace(2, 50, C.byref(size)) == 0
    if size.value:
        assert S(size=size.value - 1) == NCM_E_LENGTH and S(ws=no) == NCM_E_NULL
        assert S(ws=p + 8) == NCM_E_ARG


def test_layout(tmp_path):
    fields = kernels._SampleRules._fields_
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "ncmorph_amd.h"',
             "int main(void) {", 'printf("%zu\\n", sizeof(ncm_sample_rules_t));']
    lines += [f'printf("%zu\\n", offsetof(ncm_sample_rules_t, {f}));' for f, _ in fields]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0;", "}"]))
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o",
                    str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout
    assert [int(x) for x in out.split()] == [C.sizeof(kernels._SampleRules)] + [
        getattr(kernels._SampleRules, f).offset for f, _ in fields]
