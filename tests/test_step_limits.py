"""Sizes that the C ABI of the operators that continue a sequence refuses, on
the CPU: the pointers are never followed."""
import ctypes as C

from ncmorph_amd import kernels
from ncmorph_amd._lib import NCM_E_NULL, NCM_E_SHAPE, lib

P = 1 << 20                      # any address of enough alignment
CTX = C.c_void_p(P)


def _logits(rows=2, vocab=50, x=None, **k):
    """Its status; without logits (NULL) once all the sizes are accepted."""
    r = kernels._LogitRules(**dict(dict(requests=rows), **k))
    return lib().ncm_adjust_logits_dev(CTX, C.byref(r), x, P, rows, vocab, vocab, vocab, 0)


def test_counts_of_a_token_have_thirty_bits(ncm):
    """A token may stand in every entry of a history and every drafted row."""
    most = (1 << 30) - 1
    assert _logits(history=P, history_width=most) == NCM_E_NULL        # accepted
    assert _logits(history=P, history_width=most + 1) == NCM_E_SHAPE
    draft = dict(history=P, offsets=P, draft_tokens=P, requests=1, rows=1000)
    assert _logits(**draft, history_width=most - 1000) == NCM_E_NULL
    assert _logits(**draft, history_width=most - 999) == NCM_E_SHAPE
    assert _logits(**dict(draft, draft_tokens=None), history_width=most - 999) == NCM_E_NULL
    # Without a history its width says nothing.
    assert _logits(history_width=most + 1) == NCM_E_NULL
