"""Pages, tables and slots of a step (cache.share, cache.extend, cache.release)
against a plain list form: every entry of the tables, the stack, the holders'
counts and the step's arrays are equal."""
import numpy as np
import pytest
import torch

from ncmorph_amd import cache, kernels
from tests import step_f64 as f64

pytestmark = pytest.mark.gpu

I32 = torch.int32


class Plain:
    """The pool and the tables as lists."""

    def __init__(self, free, refs, table, page):
        self.free, self.refs = list(free), list(refs)
        self.table, self.page = [list(r) for r in table], page

    def pages(self, t):
        return min(-(-max(t, 0) // self.page), len(self.table[0]) if self.table else 0)

    def share(self, sources, tokens):
        for r, (s, t) in enumerate(zip(sources, tokens)):
            if s == r or not 0 <= s < len(self.table):
                continue
            for i in range(min(max(t, 0) // self.page, len(self.table[0]))):
                p = self.table[s][i]
                ok = 0 <= p < len(self.refs)
                self.table[r][i] = p if ok else -1
                if ok:
                    self.refs[p] += 1

    def extend(self, new, starts, rows, mask=None, take=True):
        offsets, positions, slots, missing = [0], [], [], 0
        for r, (n, s) in enumerate(zip(new, starts)):
            n, s = min(max(n, 0), rows - offsets[-1]), max(s, 0)
            if take:
                for i in range(self.pages(s), self.pages(s + n)):
                    p = self.free.pop() if self.free else -1
                    missing += p < 0
                    self.table[r][i] = p
                    if p >= 0:
                        self.refs[p] = 1
            for i in range(n):
                t = s + i
                p = self.table[r][t // self.page] if t // self.page < len(self.table[r]) else -1
                slots.append(p * self.page + t % self.page if p >= 0 else -1)
                if mask is None:
                    positions.append(t)
                else:
                    bits = [mask[offsets[-1] + i][j // 64] >> (j % 64) & 1
                            for j in range(min(n, 64 * len(mask[0])))]
                    positions.append(s + max(sum(bits) - 1, 0))
            offsets.append(offsets[-1] + n)
        positions += [0] * (rows - len(positions))
        slots += [-1] * (rows - len(slots))
        return offsets, positions, slots, missing

    def release(self, lens, keep):
        back = []
        for r, (n, k) in enumerate(zip(lens, keep)):
            n = max(n, 0)
            for i in range(self.pages(min(max(k, 0), n)), self.pages(n)):
                p, self.table[r][i] = self.table[r][i], -1
                if 0 <= p < len(self.refs):
                    back.append(p)
        held = set(p for p in back if self.refs[p] > 0)
        for p in back:
            self.refs[p] = max(self.refs[p] - 1, 0)
        gone = [p for p in dict.fromkeys(back) if self.refs[p] == 0 and p in held]
        self.free += gone[::-1]


class Both:
    """The plain form and the device's, from the same start."""

    def __init__(self, seed, requests, width, pages, page, wide=0):
        g = np.random.default_rng(seed)
        self.page = page
        free = g.permutation(pages)
        self.plain = Plain(free, [0] * pages, [[-1] * width for _ in range(requests)], page)
        self.pool = cache.PagePool(torch.from_numpy(free).to(I32).cuda(),
                                   torch.tensor([pages], dtype=I32, device="cuda"),
                                   torch.zeros(pages, dtype=I32, device="cuda"))
        # Rows of a wider table where asked for.
        self.table = torch.full((requests, width + wide), -1, dtype=I32, device="cuda")[:, :width]

    def ints(self, v):
        return torch.tensor(list(v), dtype=I32, device="cuda")

    def extend(self, new, starts, rows=None, mask=None, take=True):
        rows = sum(max(n, 0) for n in new) if rows is None else rows
        want = self.plain.extend(new, starts, rows, mask, take)
        m = None
        if mask is not None:
            m = torch.from_numpy(np.array(mask, np.uint64).reshape(rows, -1).view(np.int64)).cuda()
        got = cache.extend(self.pool if take else None, self.table, self.ints(new),
                           self.ints(starts), rows, self.page, tree_mask=m)
        assert got.offsets.tolist() == want[0]
        assert got.positions.tolist() == want[1]
        assert got.slots.tolist() == want[2]
        assert got.missing.tolist() == [want[3]]
        self.check()
        return got

    def share(self, sources, tokens):
        self.plain.share(sources, tokens)
        cache.share(self.pool, self.table, self.ints(sources), self.ints(tokens), self.page)
        self.check()

    def release(self, lens, keep):
        self.plain.release(lens, keep)
        cache.release(self.pool, self.table, self.ints(lens), self.ints(keep), self.page)
        self.check()

    def check(self):
        assert self.table.tolist() == self.plain.table
        n = int(self.pool.count)
        assert self.pool.free[:n].tolist() == self.plain.free
        assert self.pool.refs.tolist() == self.plain.refs
        assert bool((self.pool.marks == (1 << 63) - 1).all())


@pytest.mark.parametrize("requests,longest,page", [(1, 1, 16), (3, 40, 16), (48, 1, 16),
                                                   (200, 70, 32), (1500, 9, 16), (7, 3000, 64),
                                                   (1024, 4, 128), (1025, 3, 16)])
def test_rounds(cuda, requests, longest, page):
    """Steps on top of each other, some requests idle, some cut back, some done."""
    g = np.random.default_rng(requests)
    width = 5 * longest // page + 4
    b = Both(1, requests, width, requests * width, page, wide=5)
    lens = [0] * requests
    for _ in range(4):
        new = [int(g.integers(0, longest + 1)) for _ in lens]
        b.extend(new, lens, rows=sum(new) + 3)
        lens = [a + n for a, n in zip(lens, new)]
        keep = [0 if g.random() < 0.2 else a - int(g.integers(0, min(a, 20) + 1)) for a in lens]
        b.release(lens, keep)
        lens = keep


def test_release_undoes_extend(cuda):
    b = Both(2, 5, 40, 60, 16)
    b.extend([100, 0, 17, 16, 1], [0] * 5)
    before = b.pool.free.tolist(), b.pool.refs.tolist(), b.table.tolist(), int(b.pool.count)
    lens, new = [100, 0, 17, 16, 1], [30, 40, 0, 1, 15]
    after = [a + n for a, n in zip(lens, new)]
    b.extend(new, lens)
    b.release(after, lens)
    assert (b.pool.free.tolist(), b.pool.refs.tolist(), b.table.tolist(),
            int(b.pool.count)) == before


@pytest.mark.parametrize("common", [0, 15, 16, 47, 160, 5000])
def test_shared_pages(cuda, common):
    """Prefixes held by many, released in any order; the last one frees them."""
    n, width = 9, 360
    b = Both(3, n, width, 500, 16)
    b.extend([common] + [0] * (n - 1), [0] * n)
    b.share([-1, 0, 0, 99, 3, 0, -7, 0, 0], [common] * n)
    whole = common // 16 * 16
    lens = [common if r == 0 else whole if r in (1, 2, 5, 7, 8) else 0 for r in range(n)]
    new = [0, 20, 1, 5, 0, 40, 16, 3, 0]
    b.extend(new, lens)
    lens = [a + c for a, c in zip(lens, new)]
    for gone in ([0], [5, 8], [1], [2, 3, 7], [6]):
        keep = [0 if r in gone else a for r, a in enumerate(lens)]
        b.release(lens, keep)
        lens = keep
    assert int(b.pool.count) == 500 and int(b.pool.refs.sum()) == 0


def test_one_page_released_by_all_holders_at_once(cuda):
    b = Both(4, 300, 2, 5, 16)
    b.extend([32] + [0] * 299, [0] * 300)
    b.share([-1] + [0] * 299, [32] * 300)
    b.release([32] * 300, [0] * 300)
    assert int(b.pool.count) == 5


def test_entries_without_a_holder_release_nothing(cuda):
    """A page that stands in a table twice with one holder, pages that are free
    already and entries outside the pool."""
    b = Both(5, 4, 4, 20, 16)
    b.extend([64, 0, 0, 0], [0] * 4)
    for r, row in ((1, b.plain.table[0]), (2, [b.plain.free[0], 77, -3, b.plain.free[1]])):
        b.plain.table[r] = list(row)
        b.table[r] = b.ints(row)
    b.release([64] * 4, [0] * 4)
    assert int(b.pool.count) == 20


@pytest.mark.parametrize("requests", [6, 1300])
def test_pool_runs_out(cuda, requests):
    """Requests in order get pages; the tokens of the others are not there."""
    b = Both(6, requests, 6, 5, 16)
    got = b.extend([40] * requests, [0] * requests)
    assert int(got.missing) == 3 * requests - 5 and int(b.pool.count) == 0
    b.release([40] * requests, [0] * requests)
    assert int(b.pool.count) == 5


def test_lengths_out_of_range(cuda):
    """Negative lengths, tables too narrow, more tokens than rows."""
    b = Both(7, 5, 3, 30, 16)
    b.extend([-5, 100, 7, 0, 9], [-3, 0, 45, 2, 48], rows=90)
    b.extend([3, 0, 1, 0, 1], [0, 100, 52, 0, 1 << 29], rows=2)
    b.release([48, 200, -1, 1 << 30, 5], [50, 17, 0, -9, -1])


@pytest.mark.parametrize("rows,requests", [(0, 0), (5, 0), (0, 3), (5000, 0), (0, 1500)])
def test_empty_steps(cuda, rows, requests):
    b = Both(8, requests, 4, 10, 16)
    b.extend([0] * requests, [0] * requests, rows=rows)
    if requests:
        b.release([0] * requests, [0] * requests)


@pytest.mark.parametrize("requests", [4, 1100])
def test_trees(cuda, requests):
    """Positions by depth; rows in the order of the drafts."""
    new = [1 + 23 * (r % 4) for r in range(requests)]
    starts = [10 * (r % 7) for r in range(requests)]
    b = Both(9, requests, 12, 12 * requests, 16)
    b.extend(starts, [0] * requests)
    seen = f64.tree(10, new)
    rows = sum(new) + 2
    mask = f64.bits(seen, rows, 2).numpy().view(np.uint64).tolist()
    got = b.extend(new, starts, rows=rows, mask=mask)
    depth = [int(s[i].sum()) - 1 + c for s, c in zip(seen, starts) for i in range(s.shape[0])]
    assert got.positions.tolist() == depth + [0, 0]


def test_tables_that_are_there(cuda):
    """Without a pool nothing is taken; pages of any number are in the table."""
    b = Both(11, 3, 4, 12, 16)
    for r in range(3):
        row = [100 * r + 5, -1, 1 << 28, 3]
        b.plain.table[r], b.table[r] = row, b.ints(row)
    b.extend([64, 33, 2], [0, 15, 62], take=False)


def test_long_tables_and_far_slots(cuda):
    """Slots past 32 bits, a request of 60 000 tokens."""
    pool = cache.page_pool(3_000_000, "cuda")
    table = torch.full((2, 2000), -1, dtype=I32, device="cuda")
    pool.count.fill_(3_000_000)
    pool.free.copy_(torch.arange(3_000_000, device="cuda"))
    z = torch.zeros(2, dtype=I32, device="cuda")
    n = torch.tensor([60000, 1500], dtype=I32, device="cuda")
    s = cache.extend(pool, table, n, z, 61500, 1024)
    t = torch.cat([torch.arange(60000), torch.arange(1500)])
    rank = t // 1024 + torch.cat([torch.zeros(60000), torch.full((1500,), 59)]).long()
    assert torch.equal(s.slots.cpu(), (2_999_999 - rank) * 1024 + t % 1024)
    assert torch.equal(s.positions.cpu(), t.int())


def test_captured_steps(cuda):
    """A captured round of a decode loop, replayed with other lengths and eager
    work between, moves the pool as the plain form does."""
    b = Both(12, 6, 30, 100, 16)
    lens = [3, 0, 16, 40, 31, 1]
    b.extend(lens, [0] * 6)
    starts, new, keep = b.ints(lens), b.ints([0] * 6), b.ints(lens)
    total = b.ints([0] * 6)
    saved = [x.clone() for x in (b.pool.free, b.pool.count, b.pool.refs, b.table)]

    def step():
        s = cache.extend(b.pool, b.table, new, starts, 64, 16)
        torch.add(starts, new, out=total)
        cache.release(b.pool, b.table, total, keep, 16)
        return s

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for x, y in zip((b.pool.free, b.pool.count, b.pool.refs, b.table), saved):
        x.copy_(y)
    g = np.random.default_rng(13)
    for _ in range(6):
        n = [int(g.integers(0, 11)) for _ in lens]
        k = [a + int(g.integers(0, c + 1)) for a, c in zip(lens, n)]
        starts.copy_(b.ints(lens)), new.copy_(b.ints(n)), keep.copy_(b.ints(k))
        graph.replay()
        torch.cuda.synchronize()
        want = b.plain.extend(n, lens, 64)
        b.plain.release([a + c for a, c in zip(lens, n)], k)
        assert got.offsets.tolist() == want[0] and got.positions.tolist() == want[1]
        assert got.slots.tolist() == want[2]
        b.check()
        lens = k


def test_slots_are_where_write_writes(cuda):
    """The tables and offsets that extend makes drive cache.write; the cache's
    rows at the slots are the new K and V."""
    new, before = [5, 1, 0, 33], [16, 7, 3, 0]
    pool = cache.page_pool(20, "cuda")
    kv = cache.allocate(20, 2, 16, 64, torch.bfloat16, "cuda")
    table = torch.full((4, 6), -1, dtype=I32, device="cuda")
    i32 = lambda v: torch.tensor(v, dtype=I32, device="cuda")  # noqa: E731
    cache.extend(pool, table, i32(before), i32([0] * 4), sum(before), 16)
    s = cache.extend(pool, table, i32(new), i32(before), sum(new), 16)
    k, v = (torch.randn(sum(new), 128, device="cuda").to(torch.bfloat16) for _ in range(2))
    cache.write(kv, k, v, table, s.offsets, i32(before))
    got = kv.k[s.slots // 16, :, s.slots % 16].reshape(-1, 128)
    assert torch.equal(got, k)
    inv = torch.ones(32, device="cuda")
    kernels.rope_positions(k, s.positions, inv, 2, 64)  # positions are as it takes them


def test_another_stream(cuda):
    """Work goes to the current stream of the tensors' device."""
    b = Both(14, 3, 4, 12, 16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s = cache.extend(b.pool, b.table, b.ints([20, 0, 5]), b.ints([0, 0, 0]), 25, 16)
        cache.release(b.pool, b.table, b.ints([20, 0, 5]), b.ints([3, 0, 0]), 16)
    side.synchronize()
    want = b.plain.extend([20, 0, 5], [0, 0, 0], 25)
    b.plain.release([20, 0, 5], [3, 0, 0])
    assert s.slots.tolist() == want[2]
    b.check()
