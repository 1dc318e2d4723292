"""Sizes that the C ABI of the operators that continue a sequence refuses, on
the CPU: the pointers are never followed."""
import ctypes as C

from ncmorph_amd import cache, kernels
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


def _kv(**k):
    d = dict(k=P, v=P, k_scale=None, v_scale=None, k_stride=1 << 20, v_stride=1 << 20,
             k_scale_stride=0, v_scale_stride=0, pages=1, kv_heads=2, page_size=16, head_dim=64,
             codes=0)
    return C.byref(cache._Cache(**dict(d, **k)))


def _batch(**k):
    d = dict(offsets=P, starts=P, page_table=P, requests=1, rows=1, table_width=1, table_stride=1)
    return C.byref(cache._Batch(**dict(d, **k)))


def test_launches_have_32_bits_of_threads(ncm):
    """Steps of more threads than a launch can have are refused ahead of it."""
    most = 4 * ((1 << 24) - 1)                       # four rows a workgroup of 256
    for fn in (lib().ncm_kv_write_dev, lib().ncm_kv_read_dev):
        assert fn(CTX, _kv(), _batch(rows=most), None, P, 128, 128) == NCM_E_NULL
        assert fn(CTX, _kv(), _batch(rows=most + 1), None, P, 128, 128) == NCM_E_SHAPE
    size = C.c_size_t()

    def attention(rows, requests=1, heads=64):
        kv, b = _kv(kv_heads=heads), _batch(rows=rows, requests=requests)
        need = lib().ncm_kv_attention_workspace(kv, b, heads, C.byref(size))
        run = lib().ncm_kv_attention_dev(CTX, kv, b, None, P, heads, 64 * heads, 64 * heads, 1.0,
                                         0, None, None, 0, P, 1 << 60)
        return need, run

    # Units of 32 rows and one request's last: 64 of either.
    assert attention(32 * (1 << 18) - 64) == (0, NCM_E_NULL)
    assert attention(32 * (1 << 18)) == (NCM_E_SHAPE, NCM_E_SHAPE)
    # Units of up to 16 rows, one for each of many requests.
    assert attention(60000, 60000, 256) == (0, NCM_E_NULL)
    assert attention(60000, 60000, 512) == (NCM_E_SHAPE, NCM_E_SHAPE)
    # 512 threads for every row of up to 8192 float32 logits.
    most = ((1 << 32) - 1) // 512
    assert _logits(rows=most, vocab=1000) == NCM_E_NULL
    assert _logits(rows=most + 1, vocab=1000) == NCM_E_SHAPE
