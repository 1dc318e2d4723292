"""Steps that would begin inside a page with several holders (cache.extend after
cache.share and cache.release): what others read is not given as a place to
write, against the plain list form."""
import numpy as np
import pytest
import torch

from tests.test_pages_gpu import I32, Both, Plain

pytestmark = pytest.mark.gpu


class Held(Plain):
    def extend(self, new, starts, rows, mask=None, take=True):
        offsets, positions, slots, missing = super().extend(new, starts, rows, mask, take)
        for r, s in enumerate(starts):
            s, n = max(s, 0), offsets[r + 1] - offsets[r]
            at = s // self.page
            if not take or n == 0 or s % self.page == 0 or at >= len(self.table[r]):
                continue
            p = self.table[r][at]
            if 0 <= p < len(self.refs) and self.refs[p] > 1:
                missing += 1
                for i in range(min(n, (at + 1) * self.page - s)):
                    slots[offsets[r] + i] = -1
        return offsets, positions, slots, missing


def both(seed, requests, width, pages, page):
    b = Both(seed, requests, width, pages, page)
    b.plain.__class__ = Held
    return b


@pytest.mark.parametrize("requests", [4, 1100])
@pytest.mark.parametrize("keep", [15, 16, 17, 31, 32, 40, 48])
def test_cut_back_into_a_shared_page(cuda, keep, requests):
    """Holders of a common prefix, cut inside it, go on; so does its source. Once
    the others have let go the page is one's own again."""
    common, n = 48, requests
    b = both(1, n, 6, 6 * n, 16)
    b.extend([common] + [0] * (n - 1), [0] * n)
    b.share([-1, 0, 0] + [-1] * (n - 3), [common] * n)
    lens = [common] * 3 + [0] * (n - 3)
    cut = [keep if r < 2 else c for r, c in enumerate(lens)]
    b.release(lens, cut)
    new = [20, 1, 3, 7] + [0] * (n - 4)
    got = b.extend(new, cut)
    inside = keep % 16 > 0
    assert int(got.missing) == 2 * inside
    first = got.slots[:20].tolist()
    assert (first[0] < 0) == inside and first[19] >= 0
    b.release([a + c for a, c in zip(cut, new)], cut)
    # Request 2 and then 1 let the prefix go: request 0 is its last holder.
    b.release(cut, [c if r in (0, 1, 3) else 0 for r, c in enumerate(cut)])
    b.release(cut, [c if r in (0, 3) else 0 for r, c in enumerate(cut)])
    got = b.extend([20] + [0] * (n - 1), [keep] + [0] * (n - 1))
    assert int(got.missing) == 0 and -1 not in got.slots.tolist()


def test_without_a_pool_and_beside_a_dry_one(cuda):
    """The table's pages as they are where there is no pool; pages that are not
    there and pages that are others' are counted together."""
    b = both(2, 3, 4, 4, 16)
    b.extend([32, 0, 0], [0, 0, 0])
    b.share([-1, 0, 0], [32, 32, 32])
    b.extend([5, 5, 5], [20, 32, 27], take=False)
    got = b.extend([40, 5, 0], [20, 32, 32])
    assert int(got.missing) == 2                      # one page too few, one held page


def test_captured(cuda):
    """A graph of the step sees who holds what at its replay."""
    b = both(3, 3, 6, 18, 16)
    b.extend([32, 0, 0], [0] * 3)
    from ncmorph_amd import cache
    new, starts = b.ints([0, 0, 0]), b.ints([0, 0, 0])
    cache.extend(b.pool, b.table, new, starts, 30, 16)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = cache.extend(b.pool, b.table, new, starts, 30, 16)
    b.check()
    for held in (False, True, False):
        if held:
            b.share([-1, 0, -1], [32] * 3)
        for n, s in (([3, 0, 0], [20, 0, 0]), ([0, 4, 20], [0, 17 if held else 0, 0])):
            new.copy_(b.ints(n)), starts.copy_(b.ints(s))
            graph.replay()
            torch.cuda.synchronize()
            want = b.plain.extend(n, s, 30)
            assert got.offsets.tolist() == want[0] and got.positions.tolist() == want[1]
            assert got.slots.tolist() == want[2] and got.missing.tolist() == [want[3]]
            b.check()
            b.release([a + c for a, c in zip(s, n)], s)
        if held:
            b.release([0, 32, 0], [0, 0, 0])
