"""The kernel for groups of many pairs (cache.attention with groups), over runs
of several tiles: its variants of 2, 4 and 8 wavefronts of pairs, both head
sizes, all kinds of codes, with pages missing along a run and runs that cross
from one unit and group to the next. Each case says from the restated layout
what it reaches. Against 64 bits, by the bound of the attention without groups;
a request's own copy of a group's tokens holds NaN."""
import math

import pytest
import torch

from ncmorph_amd import cache
from tests import step_f64 as f64
from tests.shared_layout import WIDE_TILE, layout, up, wide_runs

pytestmark = pytest.mark.gpu

BF16, FP8, I8, I32 = torch.bfloat16, torch.float8_e4m3fn, torch.int8, torch.int32
HEADS, GROUP = 8, 8                       # K/V heads, query heads of each
PREFIXES = (4133, 3000, 3500)
MEMBERS = {2: 7, 4: 12, 8: 21}            # requests of a group that take each variant


class Batch:
    """Three groups, a request of no group, on the GPU."""

    def __init__(self, cuda, seed, members, hd, page, dtype, missing=False, blocks=1):
        self.gen = torch.Generator(device=cuda).manual_seed(seed)
        self.cuda, self.hd, self.page, self.dtype = cuda, hd, page, dtype
        self.members, self.n = members, 3 * members + 1
        self.new = [(1, 1, 2, 1, 0, 1, 1)[r % 7] for r in range(self.n)]
        # One request in ten begins ahead of its group's last shared tokens.
        self.before = []
        for r in range(self.n):
            common = PREFIXES[min(r // members, 2)]
            self.before.append(common - 70 if r % 10 == 6 else common + (r * 13) % 50)
        self.before[-1] = 77
        need = [up(c + n, page) for c, n in zip(self.before, self.new)]
        width = 32768 // page
        table = torch.full((self.n, width), -1, dtype=I32)
        at = 1                                            # page 0: NaN
        for r, k in enumerate(need):
            first = self.first(r)
            whole = 0 if r == first else min(PREFIXES[r // members], self.before[r]) // page
            table[r, :min(whole, k)] = 0
            table[r, whole:k] = torch.arange(at, at + max(k - whole, 0))
            at += max(k - whole, 0)
        self.offsets = [0]
        for n in self.new:
            self.offsets.append(self.offsets[-1] + n)
        self.rows = self.offsets[-1] + 2                  # two rows of no request
        self.layout = layout(HEADS, hd, page, self.n, self.rows, width, 3, HEADS * GROUP)
        self.done = []
        for g, common in enumerate(PREFIXES):
            mine = range(g * members, (g + 1) * members)
            pairs = sum(self.new[r] for r in mine) * GROUP
            least = min([common] + [self.before[r] for r in mine if self.new[r]])
            self.done.append((pairs, least // WIDE_TILE * WIDE_TILE))
        self.runs = wide_runs(self.layout, HEADS, self.done)
        self.missing = []                                 # (group, page of it)
        if missing:
            # A run's first, fourth, fifth and sixth tile, and one of the next.
            me = next(i for i, run in enumerate(self.runs) if i > len(self.runs) // 3
                      and len(run) >= 6 and len({(g, u) for g, u, _ in run}) == 1)
            for run, tiles in ((me, (0, 3, 4, 5)), (me + 1, (2,))):
                for t in tiles:
                    g, _, tile = self.runs[run][t]
                    p = (tile * WIDE_TILE + 17) // page
                    table[self.first(g * members), p] = (-1, 1 << 28)[t % 2]
                    self.missing.append((g, p))
        shape = (at, HEADS, page, hd)
        stores, scales, self.values = [], [], []
        for _ in range(2):
            if dtype == BF16:
                x = torch.randn(shape, generator=self.gen, device=cuda).to(BF16)
                x[0] = math.nan
                stores.append(x)
                scales.append(None)
                self.values.append(x.double())
                continue
            if dtype == FP8:
                x = torch.randn(shape, generator=self.gen, device=cuda).to(FP8)
            else:
                x = torch.randint(-127, 128, shape, generator=self.gen, device=cuda).to(I8)
            s = 0.5 + torch.rand(shape[:3], generator=self.gen, device=cuda)
            s = s if dtype == FP8 else s / 73
            s[0] = math.nan
            stores.append(x)
            scales.append(s)
            self.values.append(x.float().double() * s.double()[..., None])
        self.kv = cache.KvCache(*stores, *scales)
        self.table = table.to(cuda)
        i32 = lambda v: torch.tensor(v, dtype=I32, device=cuda)  # noqa: E731
        self.args = (self.table, i32(self.offsets), i32(self.before))
        self.groups = i32([0, members, 2 * members, 3 * members])
        self.shared = i32(PREFIXES)
        self.q = torch.randn(self.rows, HEADS * GROUP * hd, generator=self.gen, device=cuda).to(BF16)

    def first(self, r):
        return r // self.members * self.members

    def run(self, **kw):
        """The requests' rows; those of none are not initialised."""
        return cache.attention(self.q, self.kv, HEADS * GROUP, *self.args, groups=self.groups,
                               shared=self.shared, **kw)[:self.offsets[-1]]

    def check(self, got, scale=None):
        got = got.double().view(-1, HEADS, GROUP, self.hd)
        scale = self.hd ** -0.5 if scale is None else scale
        worst = 0.0
        for r in range(self.n):
            c, n, first = self.before[r], self.new[r], self.first(r)
            if n == 0:
                continue
            t = torch.arange(c + n, device=self.cuda)
            common = PREFIXES[r // self.members] if r < self.n - 1 else 0
            from_first = (t < min(common, c)) & (first != r)
            page = torch.where(from_first, self.table[first][t // self.page],
                               self.table[r][t // self.page]).long()
            there = (page >= 0) & (page < self.kv.k.shape[0])
            k, v = (x[page.clamp(0, self.kv.k.shape[0] - 1), :, t % self.page]
                    .transpose(0, 1).contiguous() for x in self.values)
            assert not bool(k[:, there].isnan().any())
            q = self.q[self.offsets[r]:self.offsets[r + 1]].double()
            q = q.view(n, HEADS, GROUP, self.hd).transpose(0, 1).reshape(HEADS, n * GROUP, self.hd)
            sees = there & (t[None] <= c + torch.arange(n, device=self.cuda)[:, None])
            sees = sees.repeat_interleave(GROUP, 0)[None]
            k, v = (torch.where(there[None, :, None], x, 0.0) for x in (k, v))
            kt = k.transpose(1, 2).contiguous()
            s = (torch.matmul(q, kt) * scale).masked_fill(~sees, -math.inf)
            p = torch.softmax(s, -1)
            ref, mag = torch.matmul(p, v), torch.matmul(p, v.abs())
            # 130 roundings of a score's products, twice their part in p.
            size = float(torch.matmul(q.abs(), kt.abs()).max()) * abs(scale)
            bound = f64.attention_bound(ref, mag) + 2 * 130 * 2.0 ** -24 * size * mag
            mine = got[self.offsets[r]:self.offsets[r + 1]].transpose(0, 1).reshape(ref.shape)
            worst = max(worst, float(((mine - ref).abs() / bound).max()))
        assert worst <= 1.0, worst

    def reaches(self, wavefronts):
        """Runs of five tiles and six, some over the borders of units and groups."""
        assert self.layout.np == wavefronts and len(self.runs) == 256
        lengths = {len(run) for run in self.runs}
        assert min(lengths) >= 5 and {x % 2 for x in lengths} == {0, 1}
        assert any(len({u for _, u, _ in run}) > 1 for run in self.runs)
        assert any(len({g for g, _, _ in run}) > 1 for run in self.runs)


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("dtype", [BF16, FP8, I8])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("wavefronts", [2, 4, 8])
def test_runs_of_tiles(cuda, wavefronts, hd, dtype, page):
    b = Batch(cuda, wavefronts + hd, MEMBERS[wavefronts], hd, page, dtype)
    b.reaches(wavefronts)
    b.check(b.run())


@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("dtype", [BF16, FP8, I8])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("wavefronts", [2, 4, 8])
def test_missing_pages_along_a_run(cuda, wavefronts, hd, dtype, page):
    b = Batch(cuda, wavefronts + hd, MEMBERS[wavefronts], hd, page, dtype, missing=True)
    b.reaches(wavefronts)
    assert len(set(b.missing)) >= (4 if page == 128 else 5)
    b.check(b.run())


@pytest.mark.parametrize("hd", [64, 128])
def test_groups_of_several_blocks(cuda, hd):
    """Forty requests a group: some 320 pairs, a block of 256 and a part of one."""
    b = Batch(cuda, hd, 40, hd, 64, BF16, missing=True)
    b.reaches(8)
    assert all(256 < pairs < 512 for pairs, _ in b.done)
    b.check(b.run())


@pytest.mark.parametrize("scale", [0.0, -0.2, 0.5])
@pytest.mark.parametrize("dtype", [BF16, FP8, I8])
@pytest.mark.parametrize("wavefronts", [2, 4, 8])
def test_scales(cuda, wavefronts, dtype, scale):
    b = Batch(cuda, 5, MEMBERS[wavefronts], 128, 64, dtype, missing=True)
    b.reaches(wavefronts)
    b.check(b.run(scale=scale), scale)


@pytest.mark.parametrize("wavefronts", [2, 4, 8])
def test_again_captured_and_on_two_streams(cuda, wavefronts):
    """Bit for bit the same each time: eagerly, in a graph that follows its
    inputs with eager work between, and where two calls run at once."""
    b = [Batch(cuda, 20 + i, MEMBERS[wavefronts], 128, 64, (BF16, FP8)[i], missing=bool(i))
         for i in range(2)]
    for x in b:
        x.reaches(wavefronts)
    want = [x.run() for x in b]
    for _ in range(3):
        assert all(torch.equal(x.run(), y) for x, y in zip(b, want))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = b[0].run()
    kept = b[0].q.clone(), b[0].shared.clone()
    for i in range(4):
        b[0].q.copy_(kept[0].roll(i, 0))
        b[0].shared.copy_(kept[1] - 64 * i)
        graph.replay()
        ref = b[0].run()
        torch.cuda.synchronize()
        assert torch.equal(got.view(torch.int16), ref.view(torch.int16))
    b[0].q.copy_(kept[0]), b[0].shared.copy_(kept[1])
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want[0])
    streams = [torch.cuda.Stream() for _ in range(2)]
    out = [[], []]
    torch.cuda.synchronize()
    for _ in range(6):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                out[i].append(b[i].run())
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in out[i])
