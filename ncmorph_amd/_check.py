"""Argument checks of the device-tensor wrappers.

The C ABI receives bare device pointers and cannot see how large each
allocation is, so a tensor of the wrong dtype or shape would be read or
written out of bounds on the GPU. Every wrapper therefore checks each tensor
argument (caller-supplied outputs included) here, before any library call,
and raises NcmError on a mismatch: dtype first, then shape, then device and
layout, so that the checks also run without a GPU.
"""
from __future__ import annotations

from ._lib import NCM_E_ARG, NCM_E_NULL, NCM_E_SHAPE, NcmError

# bf16 operands travel as 16-bit patterns: torch.bfloat16, or an int16 /
# uint16 view of the same bytes.
BF16 = ("bfloat16", "int16", "uint16")
F32 = ("float32",)
I32 = ("int32",)
U64 = ("int64", "uint64")


_NAMES = {}  # a dtype object's name, as met


def _dtype(t) -> str:
    name = _NAMES.get(t.dtype)
    if name is None:
        name = _NAMES[t.dtype] = str(t.dtype).replace("torch.", "")
    return name


class _Accepted(dict):
    """The torch dtypes that a tuple of names stands for."""

    def __missing__(self, names):
        import torch

        got = frozenset(getattr(torch, n) for n in names if hasattr(torch, n))
        self[names] = got
        return got


_ACCEPTED = _Accepted()


def _common(t, name, where, dtypes):
    if not hasattr(t, "data_ptr") or not hasattr(t, "is_cuda"):
        raise NcmError(NCM_E_ARG, where, f"{name} must be a torch tensor")
    if _dtype(t) not in dtypes:
        raise NcmError(NCM_E_ARG, where,
                       f"{name} has dtype {_dtype(t)}, expected {' or '.join(dtypes)}")


def _placed(t, name, where, device):
    if not t.is_cuda:
        raise NcmError(NCM_E_ARG, where, f"{name} must be a GPU tensor")
    if device is not None and t.device != device:
        raise NcmError(NCM_E_ARG, where, f"{name} is on {t.device}, expected {device}")


class Args:
    """The tensor arguments of one call: dev() and rows() check dtype, shape
    and layout as they are named; done() then checks that every one of them
    is a GPU tensor on the first one's device."""

    def __init__(self, where: str):
        self.where = where
        self.seen = []

    def dev(self, t, name, dtypes, shape=None, optional=False):
        """Address of a contiguous tensor of one of `dtypes` and exactly
        `shape` (None: any shape); None for an optional None."""
        W = self.where
        if t is None:
            if optional:
                return None
            raise NcmError(NCM_E_NULL, W, f"{name} is required")
        if (getattr(t, "dtype", None) in _ACCEPTED[dtypes] and t.is_contiguous()
                and (shape is None or t.shape == shape)):
            self.seen.append((t, name))  # nothing of what follows applies
            return t.data_ptr()
        _common(t, name, W, dtypes)
        if shape is not None and tuple(t.shape) != tuple(shape):
            raise NcmError(NCM_E_SHAPE, W,
                           f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
        if not t.is_contiguous():
            raise NcmError(NCM_E_ARG, W, f"{name} must be contiguous")
        self.seen.append((t, name))
        return t.data_ptr()

    def rows(self, t, name, dtypes, n_rows, min_cols):
        """(address, row stride) of a 2-D tensor with contiguous rows (a
        column slice of a wider buffer is allowed): exactly n_rows rows of
        at least min_cols elements."""
        W = self.where
        if t is None:
            raise NcmError(NCM_E_NULL, W, f"{name} is required")
        if getattr(t, "dtype", None) not in _ACCEPTED[dtypes]:
            _common(t, name, W, dtypes)
        shape = t.shape
        if len(shape) != 2 or shape[0] != n_rows or shape[1] < min_cols:
            raise NcmError(NCM_E_SHAPE, W,
                           f"{name} has shape {tuple(shape)}, expected ({n_rows}, >= {min_cols})")
        stride, inner = t.stride()
        if inner != 1 or (n_rows > 1 and stride < min_cols):
            raise NcmError(NCM_E_ARG, W, f"{name} must have contiguous, non-overlapping rows")
        self.seen.append((t, name))
        return t.data_ptr(), stride

    def done(self):
        if not self.seen:
            return
        first = self.seen[0][0]
        index = first.get_device() if first.is_cuda else -2
        for t, name in self.seen:
            if t.get_device() != index or not t.is_cuda:
                _placed(t, name, self.where, first.device)


def dims(t, name, where, ndim):
    """The shape of a tensor that must have `ndim` dimensions."""
    if t is None:
        raise NcmError(NCM_E_NULL, where, f"{name} is required")
    shape = getattr(t, "shape", None)
    if shape is None or len(shape) != ndim:
        raise NcmError(NCM_E_SHAPE, where, f"{name} must have {ndim} dimensions")
    return tuple(shape)
