"""The restated layout of the attention with groups is the library's, on the
CPU: the workspaces have the same size."""
import ctypes as C
import random

from ncmorph_amd import cache
from ncmorph_amd._lib import lib
from tests.shared_layout import layout


def test_layout(ncm):
    r = random.Random(1)
    seen = set()
    for _ in range(3000):
        heads, hd, page = r.choice([1, 2, 8, 32]), r.choice([64, 128]), r.choice([16, 64, 1024])
        q_heads = heads * r.choice([1, 2, 4, 7, 8, 24])
        requests = r.choice([1, 3, 30, 300])
        rows = r.choice([1, requests, 5 * requests, 13 * requests])
        n_groups, width = r.randint(0, min(requests, 9)), r.choice([1, 40, 500, 4000])
        kv = cache._Cache(k=1 << 20, v=1 << 20, pages=10, kv_heads=heads, page_size=page, head_dim=hd,
                       codes=0, k_stride=heads * page * hd, v_stride=heads * page * hd)
        batch = cache._Batch(offsets=1 << 20, starts=1 << 20, page_table=1 << 20,
                             requests=requests, rows=rows, table_width=width, table_stride=width)
        need = C.c_size_t()
        assert lib().ncm_kv_attention_shared_workspace(C.byref(kv), C.byref(batch), n_groups,
                                                       q_heads, C.byref(need)) == 0
        both = [layout(heads, hd, page, requests, rows, width, n_groups, q_heads, window)
                for window in (False, True)]
        assert need.value == max(s.bytes for s in both)
        seen.add(both[0].np)
    assert seen == {0, 2, 4, 8}
