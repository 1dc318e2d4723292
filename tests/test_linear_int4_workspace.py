"""linear_int4's scratch is the library's to decide, row count by row count, on
the CPU."""
import ctypes as C
from types import SimpleNamespace

import pytest
import torch

from ncmorph_amd import _check, kernels
from ncmorph_amd._lib import lib


@pytest.mark.parametrize("from_rows", [1, 2, 3, 5, 17, 65, 1 << 20])
def test_the_library_decides(ncm, monkeypatch, from_rows):
    """A library that wants scratch from `from_rows` rows on gets it."""
    real, given = lib(), []

    def workspace(m, n, k, need):
        need._obj.value = 4096 if m >= from_rows else 0
        return 0

    fake = SimpleNamespace(ncm_int4_bytes=real.ncm_int4_bytes, ncm_linear_int4_workspace=workspace,
                           ncm_linear_int4=lambda *a: given.append(a[-1]) or 0)
    monkeypatch.setattr(kernels, "lib", lambda: fake)
    monkeypatch.setattr(_check.Args, "done", lambda self: None)
    monkeypatch.setattr(kernels, "stream_context", lambda *a: SimpleNamespace(handle=None))
    w = kernels.Int4Weight(torch.zeros(1024, dtype=torch.uint8), torch.zeros(64, dtype=torch.uint8),
                           16, 128, 64, False)
    rows = [1, 2, 3, 4, 5, 16, 17, 40, 64, 65, 100]
    for m in rows:
        kernels.linear_int4(torch.zeros(m, 128, dtype=torch.bfloat16), w)
    assert given == [4096 if m >= from_rows else 0 for m in rows]


@pytest.mark.parametrize("n,k", [(0, 64), (16, 128), (256, 4096), (16385, 4096), (60000, 8)])
def test_rows_without_scratch(ncm, n, k):
    """Up to that many rows the library wants none."""
    a, b = C.c_size_t(), C.c_size_t()
    assert lib().ncm_int4_bytes(n, k, 64, 0, C.byref(a), C.byref(b)) == 0
    w = kernels.Int4Weight(torch.zeros(a.value, dtype=torch.uint8),
                           torch.zeros(b.value, dtype=torch.uint8), n, k, 64, False)
    need = C.c_size_t()
    for m in range(w.plain_rows + 1):
        assert lib().ncm_linear_int4_workspace(m, n, k, C.byref(need)) == 0 and need.value == 0
