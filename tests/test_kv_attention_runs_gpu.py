"""Attention over the paged cache where a workgroup has many tiles: steps of far
more tiles (128 tokens of a K/V head for up to 16 or 32 (row, head) pairs) than
the 512 workgroups of a launch. A run then goes from tile to tile, from unit to
unit, from one request's length to another's, and past the 32 tiles whose pages
it looks up at once. Against 64-bit softmax attention on the device, row by row.

Bound: that of tests/step_f64.py, 2^-8 of the output and 2^-10 of sum p |v|, and
the scores' rounding where they are large: hd products and sums, the two scales
and the exponent's argument are hd + 4 roundings of 2^-24 of scale * sum |q k| or
less, and an error e of the scores moves numerator and denominator of the
softmax by e each, hence the output by 2 e sum p |v|."""
import math

import pytest
import torch

from ncmorph_amd import cache
from tests import step_f64 as f64
from tests.step_f64 import BF16, FP8, I8

pytestmark = pytest.mark.gpu


class Long:
    """A step of requests with `new` rows after `before` tokens, on the device.
    growth: scores rise along the sequence, by about growth from end to end."""

    def __init__(self, cuda, seed, new, before, heads, group, hd, page, dtype, growth=0.0,
                 holes=()):
        g = torch.Generator(cuda).manual_seed(seed)
        self.new, self.before, self.heads, self.group, self.hd = new, before, heads, group, hd
        self.page, self.rows, self.holes = page, sum(new), holes
        need = [-(-(n + c) // page) for n, c in zip(new, before)]
        order = torch.randperm(sum(need) + 2, generator=g, device=cuda).int()
        self.table = torch.full((len(new), max(need) + 1), -1, dtype=torch.int32, device=cuda)
        at = 0
        for r, n in enumerate(need):
            self.table[r, :n] = order[at:at + n]
            at += n
        ends = torch.tensor([0] + new).cumsum(0)
        self.offsets = ends.int().to(cuda)
        self.starts = torch.tensor(before, dtype=torch.int32, device=cuda)
        shape = (order.numel(), heads, page, hd)
        self.values, pages, scales = [], [], []
        for which in range(2):
            # Unused places: NaN, its e4m3 code, or a NaN scale.
            p = (torch.full(shape, math.nan, dtype=BF16, device=cuda) if dtype == BF16 else
                 torch.full(shape, 127, dtype=torch.uint8, device=cuda))
            s = None if dtype == BF16 else torch.full(shape[:3], math.nan, device=cuda)
            dense = []
            for r, (n, c) in enumerate(zip(new, before)):
                t = n + c
                x = torch.randn(t, heads, hd, generator=g, device=cuda)
                if growth and which == 0:  # q has a part of one along every dim
                    x += torch.linspace(0, growth * hd ** -0.5, t, device=cuda)[:, None, None]
                if dtype == BF16:
                    codes, v = x.to(BF16), x.to(BF16).double()
                else:
                    sc = x.abs().amax(-1) / (127.0 if dtype == I8 else 400.0)
                    y = x / sc[..., None]
                    codes = y.round().to(I8) if dtype == I8 else y.to(FP8)
                    v = codes.float().double() * sc.double()[..., None]
                    codes = codes.view(torch.uint8)
                i = torch.arange(t, device=cuda)
                where = self.table[r].long()[i // page]
                p[where, :, i % page] = codes
                if s is not None:
                    s[where, :, i % page] = sc
                dense.append(v)
            self.values.append(dense)
            pages.append(p if dtype == BF16 else p.view(dtype))
            scales.append(s)
        for r, entry in holes:  # table entries of tokens that are not there
            self.table[r, entry] = -1
        self.kv = cache.KvCache(*pages, *scales)
        q = torch.randn(self.rows, heads * group * hd, generator=g, device=cuda)
        self.q = (q + 1.0 if growth else q).to(BF16)

    def tiles(self, pairs):
        return sum(self.heads * -(-n * self.group // pairs) * -(-(n + c) // 128)
                   for n, c in zip(self.new, self.before))

    def run(self, **kw):
        return cache.attention(self.q, self.kv, self.heads * self.group, self.table, self.offsets,
                               self.starts, **kw)

    def check(self, out, allowed=None, window=0):
        """allowed: per request, [n, n] pairs of new rows (None: causal)."""
        scale, group, hd, at = self.hd ** -0.5, self.group, self.hd, 0
        out = out.double().view(self.rows, self.heads, group, hd)
        q = self.q.double().view(self.rows, self.heads, group, hd)
        for r, (n, c) in enumerate(zip(self.new, self.before)):
            key = torch.arange(n + c, device=out.device)
            row = torch.arange(n, device=out.device)[:, None]
            near = key > c + row - window if window else key >= 0
            see = (key <= c + row) & near
            if allowed is not None:
                see = ((key < c) & near).expand(n, -1).clone()
                see[:, c:] = allowed[r].to(out.device)
            for rr, entry in self.holes:
                if rr == r:
                    see = see & (key // self.page != entry)
            for h in range(self.heads):
                k, v = (self.values[w][r][:, h] for w in range(2))
                x = q[at:at + n, h].reshape(n * group, hd)
                s = ((x @ k.t()) * scale).view(n, group, -1)
                size = ((x.abs() @ k.abs().t()) * scale).view(n, group, -1)
                s = s.masked_fill(~see[:, None], -math.inf)
                p = torch.softmax(s, -1).nan_to_num(0.0).view(n * group, -1)
                ref, mag = (p @ v).view(n, group, hd), (p @ v.abs()).view(n, group, hd)
                size = size.masked_fill(~see[:, None], 0.0).amax(-1, keepdim=True)
                tol = f64.attention_bound(ref, mag) + 2 * (hd + 4) * 2.0 ** -24 * size * mag
                err = (out[at:at + n, h] - ref).abs()
                assert bool((err <= tol).all()), (r, h, float((err / tol).max()))
            at += n


@pytest.mark.parametrize("dtype", [BF16, FP8, I8])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("growth", [0.0, 150.0])
def test_one_row_a_request(ncm, cuda, dtype, hd, growth):
    """16 pairs a unit, about six tiles a run; with growth, the maximum moves in
    late rounds too."""
    s = Long(cuda, 1, [1] * 7, [16000, 9001, 4095, 12345, 130, 0, 7777], 8, 2, hd, 32, dtype, growth)
    assert s.tiles(16) > 5 * 512
    s.check(s.run())


@pytest.mark.parametrize("dtype", [BF16, FP8, I8])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("growth", [0.0, 150.0])
def test_trees(ncm, cuda, dtype, hd, growth):
    """32 pairs a unit, one to three units a head of a request."""
    new = [20, 1, 33, 12]
    s = Long(cuda, 2, new, [9000, 3001, 12007, 15], 4, 2, hd, 16, dtype, growth)
    assert s.tiles(32) > 3 * 512
    seen = f64.tree(3, new)
    s.check(s.run(tree_mask=f64.bits(seen, s.rows, 1).to(cuda)), seen)


@pytest.mark.parametrize("dtype", [BF16, FP8, I8])
@pytest.mark.parametrize("hd", [64, 128])
def test_chunks(ncm, cuda, dtype, hd):
    """The causal border inside runs; the last blocks of a request not full."""
    s = Long(cuda, 3, [150, 70, 129], [4000, 2500, 0], 4, 3, hd, 64, dtype, 60.0)
    assert s.tiles(32) > 3 * 512
    s.check(s.run())


@pytest.mark.parametrize("dtype,hd,group,n", [(I8, 64, 1, 1), (BF16, 128, 4, 1), (FP8, 128, 4, 5),
                                              (I8, 128, 4, 6), (BF16, 64, 2, 9)])
@pytest.mark.parametrize("growth", [0.0, 150.0])
def test_runs_past_one_look_up(ncm, cuda, dtype, hd, group, n, growth):
    """More than 32 tiles a run, of units of more than 32 tiles."""
    before = [17500 - 3 * i for i in range(14)] + [20011, 18000]
    s = Long(cuda, 4, [n] * 16, before, 8, group, hd, 64, dtype, growth)
    assert s.tiles(16 if n * group <= 16 else 32) > 33 * 512
    s.check(s.run())


@pytest.mark.parametrize("dtype", [BF16, FP8, I8])
@pytest.mark.parametrize("n", [1, 18])
def test_holes_and_windows(ncm, cuda, dtype, n):
    """Tokens that are not there, and a window's edge, in the middle of runs."""
    before, holes = [16000, 9001, 12345, 7777], [(0, 3), (0, 400), (0, 401), (1, 100), (2, 385)]
    s = Long(cuda, 5, [n] * 4, before, 8, 2, 64, 32, dtype, 40.0, holes)
    assert s.tiles(32) > 5 * 512
    s.check(s.run())
    s.check(s.run(window=10001), window=10001)
    s = Long(cuda, 6, [n] * 4, before, 8, 2, 128, 32, dtype, 40.0, holes)
    s.check(s.run())
    s.check(s.run(window=9999), window=9999)


@pytest.mark.parametrize("dtype", [BF16, FP8, I8])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,group", [(1, 1), (1, 9), (9, 3)])
def test_many_parts(ncm, cuda, dtype, hd, n, group):
    """One unit cut into hundreds of parts."""
    s = Long(cuda, 7, [n], [40001], 1, group, hd, 64, dtype, 20.0)
    s.check(s.run())


@pytest.mark.parametrize("dtype", [BF16, FP8, I8])
def test_same_bits_again_and_captured(ncm, cuda, dtype):
    """Equal calls give equal bits; so does a captured call, replayed beside
    eager ones and with other lengths."""
    s = Long(cuda, 8, [3] * 6, [16000, 9001, 4095, 12345, 130, 7777], 8, 2, 128, 32, dtype, 80.0)
    first = s.run()
    out = torch.zeros_like(first)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.run(out=out)
    for cut in (0, 3000, 0, 4095):
        s.starts.copy_(torch.tensor([max(c - cut, 0) for c in s.before]))
        graph.replay()
        again = s.run()
        torch.cuda.synchronize()
        assert torch.equal(out, again)
        assert cut or torch.equal(again, first)
