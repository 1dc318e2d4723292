"""Attention over the cache of requests that share prefixes (cache.attention
with groups) against the plain 64-bit form, by the bound of the attention
without them. A request's own copy of what it reads through its group holds
NaN."""
import math

import numpy as np
import pytest
import torch

from ncmorph_amd import cache, kernels
from tests import step_f64 as f64

pytestmark = pytest.mark.gpu

BF16, FP8, I8, I32 = torch.bfloat16, torch.float8_e4m3fn, torch.int8, torch.int32


class Shared(f64.Step):
    """A Step whose groups' requests read their first tokens through the first
    one's row of the table."""

    def __init__(self, seed, new, before, heads, hd, page, dtype, groups, shared, **kw):
        super().__init__(seed, new, before, heads, hd, page, dtype, **kw)
        self.groups, self.shared = list(groups), list(shared)
        raw = torch.uint8 if dtype != BF16 else BF16
        for g, common in enumerate(shared):
            first, last = groups[g], groups[g + 1]
            for r in range(first + 1, last):
                n = min(common, before[r])
                for dense, pages, scales in zip(self.tokens, self.pages, self.scales):
                    dense[r][:n] = dense[first][:n]
                    for t in range(n):
                        p = int(self.table[r, t // page])
                        pages.view(raw)[p, :, t % page] = 127 if dtype != BF16 else math.nan
                        if scales is not None:
                            scales[p, :, t % page] = math.nan

    def run(self, cuda, q, q_heads, **kw):
        kv, table, offsets, starts = self.to(cuda)
        i32 = lambda v: torch.tensor(v, dtype=I32, device=cuda)  # noqa: E731
        return cache.attention(q, kv, q_heads, table, offsets, starts, groups=i32(self.groups),
                               shared=i32(self.shared), **kw)


def queries(seed, rows, width):
    return torch.randn(rows, width, generator=torch.Generator().manual_seed(seed)).to(BF16)


def close(got, ref, mag, rows=None):
    got = got.double().cpu().view(ref.shape)
    there = ~ref.isnan()
    err, bound = (got - ref).abs(), f64.attention_bound(ref, mag)
    assert bool((err <= bound)[there].all()), float((err / bound)[there].max())


CASES = [
    # new rows, tokens before, groups, shared
    ([1, 1], [40, 40], [0, 2], [32]),
    ([1, 1, 1, 1], [300, 257, 290, 400], [0, 4], [256]),
    ([1] * 6, [130, 129, 140, 128, 500, 135], [0, 6], [127]),          # in no whole page
    ([1] * 5, [20, 3, 9, 17, 5], [0, 5], [17]),                        # more than some have
    ([1, 2, 5, 1, 3], [200, 100, 150, 90, 0], [0, 2, 5], [95, 80]),    # one has nothing before
    ([3, 1, 1, 4, 1, 1, 2], [64, 48, 70, 33, 50, 49, 200], [1, 4, 6], [33, 1]),  # not all grouped
    ([1, 1, 1], [100, 100, 100], [0, 1, 3], [64, 0]),                  # alone, and nothing shared
    ([1] * 40, [1000] + [970 + i for i in range(39)], [0, 40], [960]),
    ([17, 0, 30, 9], [600, 500, 555, 520], [0, 4], [500]),             # one without rows
    ([40, 25], [700, 640], [0, 2], [630]),
]


@pytest.mark.parametrize("dtype", [BF16, FP8, I8])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_groups(cuda, dtype, case):
    new, before, groups, shared = CASES[case]
    hd, page = (64, 128)[case % 2], (16, 32, 64)[case % 3]
    heads, q_heads = ((2, 8), (1, 3), (4, 4))[case % 3]
    s = Shared(case, new, before, heads, hd, page, dtype, groups, shared, extra_rows=2)
    q = queries(case, s.rows, q_heads * hd)
    ref, mag = f64.attention(s, q, q_heads, f64.chain(new), chained=True)
    close(s.run(cuda, q.to(cuda), q_heads), ref, mag)


@pytest.mark.parametrize("dtype", [BF16, FP8])
@pytest.mark.parametrize("hd", [64, 128])
def test_trees(cuda, hd, dtype):
    new, before = [13, 7, 1, 30, 70], [200, 190, 300, 180, 181]
    s = Shared(1, new, before, 2, hd, 16, dtype, [0, 3, 5], [185, 170])
    seen = f64.tree(2, new)
    seen[0][4] = False                                    # sees no new token
    mask = f64.bits(seen, s.rows, 2)
    q = queries(3, s.rows, 6 * hd)
    ref, mag = f64.attention(s, q, 6, seen)
    close(s.run(cuda, q.to(cuda), 6, tree_mask=mask.to(cuda)), ref, mag)


@pytest.mark.parametrize("window", [1, 50, 100, 100000])
@pytest.mark.parametrize("given", [False, True])
def test_windows(cuda, window, given):
    """Windows that end inside the prefix, behind it, or reach past it."""
    new, before = [1, 4, 1, 3], [700, 300, 310, 340]
    s = Shared(4, new, before, 2, 64, 16, BF16, [0, 4], [290])
    positions = None
    if given:
        positions = torch.tensor([c + 3 * i for n, c in zip(new, before) for i in range(n)],
                                 dtype=I32)
    q = queries(5, s.rows, 256)
    if given:
        seen = f64.tree(6, new)
        ref, mag = f64.attention(s, q, 4, seen, window=window, positions=positions)
        got = s.run(cuda, q.to(cuda), 4, window=window, positions=positions.to(cuda),
                    tree_mask=f64.bits(seen, s.rows, 1).to(cuda))
    else:
        ref, mag = f64.attention(s, q, 4, f64.chain(new), window=window, chained=True)
        got = s.run(cuda, q.to(cuda), 4, window=window)
    close(got, ref, mag)


class Roomy(Shared):
    """A table with room for so many tokens that groups of many pairs take the
    kernel that is theirs, 2^31 (row, head) pairs x tokens x head_dim."""

    def to(self, cuda):
        kv, table, offsets, starts = super().to(cuda)
        page = kv.k.shape[2]
        width = 2 ** 31 // (self.rows * self.q_heads * kv.k.shape[3] * page) + 1
        more = torch.full((table.shape[0], max(width, table.shape[1])), -1, dtype=I32, device=cuda)
        more[:, :table.shape[1]] = table
        return kv, more, offsets, starts

    def run(self, cuda, q, q_heads, **kw):
        self.q_heads = q_heads
        return super().run(cuda, q, q_heads, **kw)


@pytest.mark.parametrize("dtype", [BF16, FP8, I8])
@pytest.mark.parametrize("share", [16, 40])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_groups_of_many_pairs(cuda, case, share, dtype):
    """Sixteen or forty heads a K/V head: 16 to 1040 pairs a group."""
    new, before, groups, shared = CASES[case]
    hd, page, heads = (64, 128)[case % 2], (16, 32, 64)[case % 3], 1 + case % 2
    s = Roomy(60 + case, new, before, heads, hd, page, dtype, groups, shared, extra_rows=2)
    q = queries(case, s.rows, heads * share * hd)
    ref, mag = f64.attention(s, q, heads * share, f64.chain(new), chained=True)
    close(s.run(cuda, q.to(cuda), heads * share), ref, mag)


@pytest.mark.parametrize("dtype", [BF16, FP8])
@pytest.mark.parametrize("hd", [64, 128])
def test_trees_of_many_pairs(cuda, hd, dtype):
    new, before = [13, 7, 1, 30, 70], [200, 190, 300, 180, 181]
    s = Roomy(71, new, before, 2, hd, 16, dtype, [0, 3, 5], [185, 170])
    seen = f64.tree(72, new)
    mask = f64.bits(seen, s.rows, 2)
    q = queries(73, s.rows, 16 * hd)
    ref, mag = f64.attention(s, q, 16, seen)
    close(s.run(cuda, q.to(cuda), 16, tree_mask=mask.to(cuda)), ref, mag)


def test_missing_pages_and_infinities_of_many_pairs(cuda):
    """A page that is not there, and an infinity among the values, in a prefix
    that the kernel for many pairs reads."""
    new, before = [1] * 6, [200, 180, 190, 200, 185, 199]
    s = Roomy(74, new, before, 1, 64, 16, BF16, [0, 6], [176])
    s.table[0, 3] = -1                                    # tokens 48 .. 63
    s.tokens[1][0][100, 0, 5] = math.inf
    p = int(s.table[0, 100 // 16])
    s.pages[1][p, 0, 100 % 16, 5] = math.inf
    q = queries(75, s.rows, 24 * 64)
    got = s.run(cuda, q.to(cuda), 24).float().cpu().view(6, 24, 64)
    assert bool((got[..., 5] == math.inf).all())
    for r, c in enumerate(before):
        at = [i for i in range(c + 1) if not 48 <= i < 64]
        there = lambda x: torch.cat([x[0][:176], x[r][176:]])[at][:, 0].double()  # noqa: E731
        k, v = there(s.tokens[0]), there(s.tokens[1])
        v[:, 5] = 0
        w = torch.softmax(q[r].view(24, 64).double() @ k.t() / 8, 1)
        rest = got[r].double().clone()
        rest[:, 5] = 0
        assert bool(((rest - w @ v).abs() <= f64.attention_bound(w @ v, w @ v.abs())).all())


def test_missing_pages(cuda):
    """A page that the first request's row lacks is not there for the group; one
    that its own row lacks is not for a request."""
    new, before = [1, 1, 1], [100, 90, 95]
    s = Shared(7, new, before, 2, 64, 16, BF16, [0, 3], [80])
    s.table[0, 2], s.table[1, 5] = -1, 1 << 20
    missing = [(r, 2) for r in range(3)] + [(1, 5)]
    q = queries(8, s.rows, 256)
    ref, mag = f64.attention(s, q, 4, f64.chain(new), missing=missing, chained=True)
    close(s.run(cuda, q.to(cuda), 4), ref, mag)
    s.table[:] = -1
    assert float(s.run(cuda, q.to(cuda), 4).abs().max()) == 0.0


@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
@pytest.mark.parametrize("dtype", [BF16, I8])
def test_scales_and_large_scores(cuda, scale, dtype):
    new, before = [1, 2, 1], [300, 280, 290]
    s = Shared(9, new, before, 2, 128, 16, dtype, [0, 3], [273])
    q = queries(10, s.rows, 4 * 128)
    ref, mag = f64.attention(s, q, 4, f64.chain(new), scale=scale, chained=True)
    # Scores of up to 2 * 128 * 9, the error of their 130 roundings times the
    # probabilities: 130 * 2^-24 * 2300 = 2^-5.8 at most; here a row's largest
    # sum |q k| scale is below 500.
    got = s.run(cuda, q.to(cuda), 4, scale=scale).double().cpu().view(ref.shape)
    bound = f64.attention_bound(ref, mag) + 130 * 2.0 ** -24 * 500 * 2 * mag
    assert bool(((got - ref).abs() <= bound).all())


def test_values_that_are_not_finite(cuda):
    """Infinities and NaN among the shared values reach those that see them, and
    no row of a request that does not hold the token."""
    new, before = [1, 1, 1, 1], [64, 20, 64, 64]
    s = Shared(11, new, before, 1, 64, 16, BF16, [0, 3], [48])
    s.tokens[1][0][30, 0, 5] = math.inf
    for r in (1, 2):
        s.tokens[1][r][:min(48, before[r])] = s.tokens[1][0][:min(48, before[r])]
    p = int(s.table[0, 30 // 16])
    s.pages[1][p, 0, 30 % 16, 5] = math.inf
    q = queries(12, s.rows, 128)
    got = s.run(cuda, q.to(cuda), 2).float().cpu().view(4, 2, 64)
    assert bool((got[0, :, 5] == math.inf).all()) and bool((got[2, :, 5] == math.inf).all())
    rest = got.clone()
    rest[0, :, 5] = rest[2, :, 5] = 0
    assert bool(torch.isfinite(rest).all())


def test_in_place_and_strided(cuda):
    """out = q, queries as columns of a wider buffer."""
    new, before = [2, 1, 1, 3], [150, 140, 139, 160]
    s = Shared(13, new, before, 2, 64, 32, FP8, [0, 4], [128], extra_rows=1)
    wide = queries(14, s.rows, 512 + 16)
    q = wide[:, 8:8 + 512]
    ref, mag = f64.attention(s, q, 8, f64.chain(new), chained=True)
    dev = wide.to(cuda)
    view = dev[:, 8:8 + 512]
    got = s.run(cuda, view, 8, out=view)
    close(got, ref, mag)
    assert torch.equal(dev[:, :8].cpu(), wide[:, :8]) and torch.equal(dev[:, 520:].cpu(), wide[:, 520:])
    assert torch.equal(dev[-1].cpu(), wide[-1])           # a row of no request


def test_many_pairs_and_long_prefixes(cuda):
    """Prefixes cut into many runs; groups whose pairs fill several blocks. One
    request of the group alone gives the same within both sums' bounds."""
    n, common, hd = 90, 5952, 128
    g = torch.Generator().manual_seed(15)
    pages = common // 64 + n + 1
    kv = cache.KvCache(*(torch.randn(pages, 2, 64, hd, generator=g).to(BF16).to(cuda)
                         for _ in range(2)))
    table = torch.full((n, common // 64 + 2), -1, dtype=I32)
    table[:, :common // 64] = torch.arange(common // 64)
    table[:, common // 64] = common // 64 + torch.arange(n)
    table = table.to(cuda)
    before = torch.tensor([common // 64 * 64 + i % 63 for i in range(n)], dtype=I32, device=cuda)
    offsets = torch.arange(n + 1, dtype=I32, device=cuda)
    q = queries(16, n, 8 * hd).to(cuda)
    i32 = lambda *v: torch.tensor(v, dtype=I32, device=cuda)  # noqa: E731
    plain = cache.attention(q, kv, 8, table, offsets, before)
    for groups, shared in ((i32(0, n), i32(common)), (i32(0, 30, 31, 80), i32(common, 64, 5000)),
                           (i32(), None)):
        if shared is None:
            groups, shared = i32(0), i32()
        got = cache.attention(q, kv, 8, table, offsets, before, groups=groups, shared=shared)
        # Both are within 2^-10 sum p |v| + 2^-8 |o| of the exact value; |v| < 6.
        bound = 2 * (2.0 ** -10 * 6 + 2.0 ** -8 * plain.float().abs())
        assert bool(((got.float() - plain.float()).abs() <= bound).all())


def test_captured(cuda):
    """A graph follows groups, lengths and tables at replay, bit for bit as the
    eager call, with eager work between."""
    new, before = [1, 2, 1, 1], [200, 180, 190, 170]
    s = Shared(17, new, before, 2, 64, 16, BF16, [0, 4], [160])
    kv, table, offsets, starts = s.to(cuda)
    groups = torch.tensor([0, 2, 4], dtype=I32, device=cuda)
    shared = torch.tensor([0, 0], dtype=I32, device=cuda)
    q = queries(18, s.rows, 512).to(cuda)
    args = (q, kv, 8, table, offsets, starts)
    cache.attention(*args, groups=groups, shared=shared)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = cache.attention(*args, groups=groups, shared=shared)
    for a, b in (([0, 4, 4], [160, 9]), ([0, 0, 4], [7, 100]), ([0, 4, 4], [160, 0])):
        groups.copy_(torch.tensor(a)), shared.copy_(torch.tensor(b))
        graph.replay()
        ref = cache.attention(*args, groups=groups, shared=shared)
        torch.cuda.synchronize()
        assert torch.equal(got.view(torch.int16), ref.view(torch.int16))
        assert torch.isfinite(got.float()).all() == (a != [0, 0, 4])  # its own copy holds NaN
    want, mag = f64.attention(s, q.cpu(), 8, f64.chain(new), chained=True)
    shared.copy_(torch.tensor([160, 0])), groups.copy_(torch.tensor([0, 4, 4]))
    graph.replay()
    torch.cuda.synchronize()
    close(got, want, mag)


def test_two_streams(cuda):
    """Two calls at once, each with a workspace of its own."""
    steps = [Shared(20 + i, [1] * 5, [400, 390, 380, 399, 398], 2, 64, 16, BF16, [0, 5], [370])
             for i in range(2)]
    qs = [queries(30 + i, 5, 256).to(cuda) for i in range(2)]
    on = [s.to(cuda) for s in steps]
    g = torch.tensor([0, 5], dtype=I32, device=cuda)
    c = torch.tensor([370], dtype=I32, device=cuda)
    call = lambda i: cache.attention(qs[i], on[i][0], 4, *on[i][1:], groups=g, shared=c)  # noqa
    want = [call(i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(call(i))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_step_of_a_batch(cuda):
    """What one decode step runs, together: pages shared and taken, positions and
    slots, rotation, the cache, attention over the common prefix, a 4-bit output
    projection, rules on the logits and the draw; every stage against its plain
    form on that stage's input."""
    n, common, hd, qh, kh, vocab = 6, 100, 64, 4, 2, 500
    g = torch.Generator().manual_seed(40)
    pool = cache.page_pool(60, cuda)
    kv = cache.allocate(60, kh, 16, hd, BF16, cuda)
    table = torch.full((n, 12), -1, dtype=I32, device=cuda)
    i32 = lambda v: torch.tensor(v, dtype=I32, device=cuda)  # noqa: E731
    rand = lambda *s: torch.randn(*s, generator=g).to(BF16).to(cuda)  # noqa: E731
    zero = i32([0] * n)
    # The prompt, by the first request; the others hold its whole pages.
    s = cache.extend(pool, table, i32([common] + [0] * (n - 1)), zero, common, 16)
    k0, v0 = rand(common, kh * hd), rand(common, kh * hd)
    cache.write(kv, k0, v0, table, s.offsets, zero)
    cache.share(pool, table, i32([-1] + [0] * (n - 1)), i32([common] * n), 16)
    starts = [common] + [96] * (n - 1)
    dense_k = [k0.cpu()[:c] for c in starts]
    dense_v = [v0.cpu()[:c] for c in starts]
    inv = torch.ones(hd // 2, device=cuda) * 0.1
    codes, scales, _ = kernels.quantise_int4(rand(vocab, qh * hd), 64)
    head = kernels.pack_int4(codes, scales, 64)
    w = (codes.cpu().double() - 8) * scales.cpu().double().repeat_interleave(64, 1)
    groups, shared = i32([0, n]), i32([96])
    for turn in range(5):
        new = [1] * n if turn else [1, 3, 5, 1, 20, 2]
        rows = sum(new)
        s = cache.extend(pool, table, i32(new), i32(starts), rows, 16)
        assert int(s.missing) == 0
        at = [c + i for c, m in zip(starts, new) for i in range(m)]
        assert s.positions.tolist() == at
        q, k, v = rand(rows, qh * hd), rand(rows, kh * hd), rand(rows, kh * hd)
        q = kernels.rope_positions(q, s.positions, inv, qh, hd)
        k = kernels.rope_positions(k, s.positions, inv, kh, hd)
        cache.write(kv, k, v, table, s.offsets, i32(starts))
        o = cache.attention(q, kv, qh, table, s.offsets, i32(starts), groups=groups, shared=shared)
        off = s.offsets.tolist()
        for r in range(n):
            dense_k[r] = torch.cat([dense_k[r], k.cpu()[off[r]:off[r + 1]]])
            dense_v[r] = torch.cat([dense_v[r], v.cpu()[off[r]:off[r + 1]]])
            for i in range(new[r]):
                for h in range(qh):
                    end = starts[r] + i + 1
                    kk, vv = (x[r][:end].view(end, kh, hd)[:, h // 2].double()
                              for x in (dense_k, dense_v))
                    p = torch.softmax(kk @ q.cpu()[off[r] + i].view(qh, hd)[h].double() / 8, 0)
                    got = o[off[r] + i].view(qh, hd)[h].double().cpu()
                    bound = f64.attention_bound(p @ vv, p @ vv.abs())
                    assert bool(((got - p @ vv).abs() <= bound).all())
        logits = kernels.linear_int4(o, head)
        x = o.cpu().double()
        e = x.abs() @ (torch.full_like(w, 280.0) * scales.cpu().double().abs()
                       .repeat_interleave(64, 1)).t()
        assert bool(((logits.cpu().double() - x @ w.t()).abs() <= 150 * 2.0 ** -24 * e).all())
        logits = kernels.adjust_logits(logits, offsets=s.offsets,
                                       bias_ids=i32([[7]] * n),
                                       bias_values=torch.full((n, 1), 3.0, device=cuda))
        u = torch.rand(rows, generator=g).to(cuda)
        top_p = torch.full((n,), 0.8, device=cuda)
        token = kernels.sample(logits, u, top_p=top_p, offsets=s.offsets).cpu()
        for i in range(rows):
            z = logits[i].cpu().double()
            order = torch.argsort(z, descending=True, stable=True)
            p = torch.softmax(z[order], 0)
            c = p.cumsum(0)
            kept = int((c < float(top_p[0])).sum()) + 1
            j = int((c[:kept] <= float(u[i].double()) * float(c[kept - 1])).sum())
            assert int(token[i]) == int(order[j])
        lens = [c + m for c, m in zip(starts, new)]
        starts = [c + 1 for c in starts]                   # one token is accepted
        cache.release(pool, table, i32(lens), i32(starts), 16)
        dense_k = [x[:c] for x, c in zip(dense_k, starts)]
        dense_v = [x[:c] for x, c in zip(dense_v, starts)]
    cache.release(pool, table, i32(starts), zero, 16)
    assert int(pool.count) == 60 and int(pool.refs.sum()) == 0
