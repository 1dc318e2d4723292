"""Attention over the paged cache against 64-bit softmax attention of what the
cache stands for, within the bound that tests/step_f64.py derives. Unused
places of the cache hold NaN."""
import math

import numpy as np
import pytest
import torch

from ncmorph_amd import cache
from ncmorph_amd._lib import NcmError
from tests import step_f64 as f64
from tests.step_f64 import BF16, FP8, I8

pytestmark = pytest.mark.gpu

DTYPES = [BF16, FP8, I8]


def queries(step, q_heads, cuda, seed=5, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(step.rows, q_heads * step.hd, generator=g) * std).to(BF16).to(cuda)


def held(out, step, q_heads, ref, mag):
    out = out.cpu().double().reshape(step.rows, q_heads, step.hd)
    n = sum(step.new)
    err, tol = (out - ref).abs()[:n], f64.attention_bound(ref, mag)[:n]
    assert bool((err <= tol).all()), float((err / tol).max())


def run(step, q_heads, cuda, allowed=None, words=None, **kw):
    q = queries(step, q_heads, cuda)
    kv, table, offs, starts = step.to(cuda)
    mask = None if allowed is None else f64.bits(allowed, step.rows, words).to(cuda)
    pos = kw.get("positions")
    out = cache.attention(q, kv, q_heads, table, offs, starts, tree_mask=mask,
                          **dict(kw, positions=None if pos is None else pos.to(cuda)))
    return q.cpu(), out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd,q_heads,heads", [(64, 3, 1), (64, 14, 2), (128, 8, 2), (128, 2, 2),
                                              (64, 40, 1)])
@pytest.mark.parametrize("before,page", [([0], 16), ([1, 0, 15], 16), ([16, 31, 32, 33], 16),
                                         ([127, 128, 129, 400], 64), ([700, 3], 256)])
def test_one_token(ncm, cuda, dtype, hd, q_heads, heads, before, page):
    step = f64.Step(1, [1] * len(before), before, heads, hd, page, dtype)
    q, out = run(step, q_heads, cuda)
    held(out, step, q_heads, *f64.attention(step, q, q_heads, f64.chain(step.new)))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd,q_heads,heads", [(64, 4, 2), (128, 4, 1), (128, 2, 2)])
@pytest.mark.parametrize("new,before", [
    ([2], [0]), ([5, 0, 1, 17], [40, 9, 0, 127]), ([25, 24], [100, 0]), ([65], [70]),
    ([33, 64, 1], [31, 128, 250])])
def test_trees(ncm, cuda, dtype, hd, q_heads, heads, new, before):
    step = f64.Step(2, new, before, heads, hd, 16, dtype, extra_rows=3)
    allowed = f64.tree(4, new)
    q, out = run(step, q_heads, cuda, allowed, (max(new) + 63) // 64)
    held(out, step, q_heads, *f64.attention(step, q, q_heads, allowed))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd,q_heads,heads,new,before", [
    (64, 2, 1, [150], [0]), (128, 4, 2, [40, 90], [50, 0]), (128, 1, 1, [200], [77])])
def test_chunks(ncm, cuda, dtype, hd, q_heads, heads, new, before):
    step = f64.Step(3, new, before, heads, hd, 32, dtype)
    q, out = run(step, q_heads, cuda)
    held(out, step, q_heads, *f64.attention(step, q, q_heads, f64.chain(new)))


@pytest.mark.parametrize("window", [1, 7, 33, 1000])
@pytest.mark.parametrize("form", ["one", "chain", "tree"])
def test_windows(ncm, cuda, window, form):
    new, before = ([1, 1, 1], [300, 20, 0]) if form == "one" else ([20, 3, 9], [300, 20, 0])
    step = f64.Step(6, new, before, 2, 64, 16, FP8)
    allowed = f64.tree(8, new) if form == "tree" else f64.chain(new)
    pos = None
    if form == "tree":       # positions by depth; one below its request's start
        pos = torch.cat([a.sum(1).int() - 1 + c for a, c in zip(allowed, before)])
        pos[3] = -5
        pos = pos.int()
    q, out = run(step, 6, cuda, allowed if form == "tree" else None, 1, window=window,
                 positions=pos)
    held(out, step, 6, *f64.attention(step, q, 6, allowed, window=window, positions=pos,
                                      chained=form != "tree"))


def test_rows_that_see_nothing(ncm, cuda):
    """Empty masks over an empty context, and a window that leaves nothing, are
    zeros; masks may leave the row itself out, or set bits past the request."""
    new, before = [4, 3], [0, 5]
    step = f64.Step(9, new, before, 1, 64, 16, BF16)
    allowed = [torch.zeros(4, 4).bool(), torch.zeros(3, 3).bool()]
    allowed[0][1, 3] = True
    mask = f64.bits(allowed, 7, 1)
    mask[2, 0] = -16                    # bits 4 .. 63: no rows of that request
    q = queries(step, 2, cuda)
    kv, table, offs, starts = step.to(cuda)
    out = cache.attention(q, kv, 2, table, offs, starts, tree_mask=mask.to(cuda))
    held(out, step, 2, *f64.attention(step, q.cpu(), 2, allowed))
    assert float(out[[0, 2, 3]].abs().max()) == 0.0 and float(out[1].abs().max()) > 0.0
    far = torch.tensor([0, 0, 0, 0, 900, 901, 902], dtype=torch.int32, device=cuda)
    out = cache.attention(q, kv, 2, table, offs, starts, tree_mask=mask.to(cuda) * 0, window=10,
                          positions=far)
    assert float(out.abs().max()) == 0.0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_what_is_not_seen_does_not_reach_a_row(ncm, cuda, dtype, value):
    """K and V of one drafted token and of one token that only a window hides
    hold a value that is not finite: the rows that see neither are as without."""
    new, before = [6], [40]
    step = f64.Step(10, new, before, 1, 64, 16, dtype)
    allowed = [torch.eye(6).bool() | torch.tensor([[True] + [False] * 5])]
    allowed[0][5, 4] = True             # row 5 and row 4 see token 4
    ref, mag = f64.attention(step, torch.zeros(6, 128), 2, allowed)
    q = queries(step, 2, cuda)
    pos = torch.tensor([40, 41, 41, 41, 41, 62], dtype=torch.int32)
    ref, mag = f64.attention(step, q.cpu(), 2, allowed, window=30, positions=pos)
    for which in (0, 1):
        bad = f64.Step(10, new, before, 1, 64, 16, dtype)
        for t in (12, 44):              # 12: hidden from row 5 alone (62 - 30 = 32)
            p, at = int(bad.table[0, t // 16]), t % 16
            if dtype == BF16:
                bad.pages[which][p, 0, at, 3] = value
            else:
                codes, sc = f64.quantise(torch.full((1, 64), value).to(BF16), dtype)
                bad.pages[which][p, 0, at] = codes[0]
                bad.scales[which][p, 0, at] = sc[0]
        kv, table, offs, starts = bad.to(cuda)
        mask = f64.bits(allowed, 6, 1).to(cuda)
        # Only token 44 is bad for rows that see all the context.
        p, at = int(step.table[0, 0]), 12
        good, table2, offs, starts = step.to(cuda)
        for w in range(2):
            dst, src = ((good.k, kv.k), (good.v, kv.v))[w]
            p44 = int(step.table[0, 2])
            dst.view(torch.uint8)[p44, 0, 44 % 16] = src.view(torch.uint8)[p44, 0, 44 % 16]
            if dtype != BF16:
                (good.k_scale, good.v_scale)[w][p44, 0, 44 % 16] = (
                    kv.k_scale, kv.v_scale)[w][p44, 0, 44 % 16]
        out = cache.attention(q, good, 2, table, offs, starts, tree_mask=mask, window=30,
                              positions=pos.to(cuda))
        o = out.cpu().double().reshape(6, 2, 64)
        seeing = torch.tensor([4, 5])
        for i in range(4):
            assert bool(((o[i] - ref[i]).abs() <= f64.attention_bound(ref, mag)[i]).all())
        if which == 1 and dtype == BF16:   # the column of the bad value, and no other
            col = o[seeing][..., 3]
            assert bool(torch.isnan(col).all()) if math.isnan(value) else bool((col == value).all())
            rest = torch.arange(64) != 3
            assert bool(torch.isfinite(o[seeing][..., rest]).all())
        elif which == 1 or math.isnan(value) or dtype != BF16:
            assert bool(torch.isnan(o[seeing]).all())
        # Token 12 too: row 5's window leaves it out, rows 0 .. 4 see it.
        out = cache.attention(q, kv, 2, table, offs, starts, tree_mask=mask & ~(1 << 4),
                              window=30, positions=pos.to(cuda))
        o = out.cpu().double().reshape(6, 2, 64)
        seen = allowed[0].clone()
        seen[:, 4] = False
        ref2, mag2 = f64.attention(step, q.cpu(), 2, [seen], window=30, positions=pos)
        assert bool(((o[5] - ref2[5]).abs() <= f64.attention_bound(ref2, mag2)[5]).all())


def test_infinities_of_both_signs(ncm, cuda):
    """V of two drafted tokens +inf and -inf in one column: each alone gives
    its infinity, both NaN; neither, a number."""
    step = f64.Step(12, [4], [3], 1, 64, 16, BF16)
    for t, value in ((4, math.inf), (5, -math.inf)):
        step.pages[1][int(step.table[0, 0]), 0, t, 7] = value
    allowed = torch.tensor([[1, 0, 0, 0], [0, 1, 0, 0], [0, 0, 1, 0], [0, 1, 1, 1]]).bool()
    q = queries(step, 1, cuda)
    kv, table, offs, starts = step.to(cuda)
    o = cache.attention(q, kv, 1, table, offs, starts,
                        tree_mask=f64.bits([allowed], 4, 1).to(cuda)).cpu()
    assert math.isfinite(o[0, 7]) and o[1, 7] == math.inf and o[2, 7] == -math.inf
    assert math.isnan(o[3, 7])
    rest = torch.arange(64) != 7
    assert bool(torch.isfinite(o[:, rest]).all())


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("before", [0, 200])
def test_values_that_are_not_finite_where_all_see_them(ncm, cuda, value, before):
    """The column of the value holds it, the others what they would without."""
    step = f64.Step(22, [1, 3], [before, 70], 1, 64, 16, BF16)
    q = queries(step, 2, cuda)
    ref, mag = f64.attention(step, q.cpu(), 2, f64.chain(step.new))
    for r in range(2):
        step.pages[1][int(step.table[r, 0]), 0, 0, 5] = value
    kv, table, offs, starts = step.to(cuda)
    o = cache.attention(q, kv, 2, table, offs, starts).cpu().double().reshape(4, 2, 64)
    col = o[..., 5]
    assert bool(torch.isnan(col).all()) if math.isnan(value) else bool((col == value).all())
    rest = torch.arange(64) != 5
    err, tol = (o - ref).abs()[..., rest], f64.attention_bound(ref, mag)[..., rest]
    assert bool((err <= tol).all())


@pytest.mark.parametrize("scale", [0.0, 0.5, 3.0, -0.5])
def test_scales_and_large_scores(ncm, cuda, scale):
    """Scores of hundreds: one token carries the softmax. Their fp32 rounding,
    2^-24 of the score per product and sum, moves a probability by as much:
    130 * 2^-24 * |s| with |s| <= 3 * 64 * 10 * 5, added to the bound."""
    step = f64.Step(13, [1, 3], [200, 40], 2, 64, 16, BF16)
    q = queries(step, 4, cuda, std=10.0)
    kv, table, offs, starts = step.to(cuda)
    out = cache.attention(q, kv, 4, table, offs, starts, scale=scale)
    ref, mag = f64.attention(step, q.cpu(), 4, f64.chain(step.new), scale=scale)
    out = out.cpu().double().reshape(ref.shape)
    tol = f64.attention_bound(ref, mag) + 130 * 2.0 ** -24 * abs(scale) * 3200 * mag
    assert bool(((out - ref).abs() <= tol).all())


def test_pages_that_are_not_there(ncm, cuda):
    """Entries outside the cache hide their tokens, wherever they lie."""
    step = f64.Step(14, [3, 1], [100, 64], 1, 64, 16, FP8)
    kv, table, offs, starts = step.to(cuda)
    q = queries(step, 2, cuda)
    table[0, 2], table[0, 3], table[1, 0] = -1, step.pages[0].shape[0], 2**31 - 1
    out = cache.attention(q, kv, 2, table, offs, starts)
    held(out, step, 2, *f64.attention(step, q.cpu(), 2, f64.chain(step.new),
                                      missing=[(0, 2), (0, 3), (1, 0)]))
    # A table that ends early, and one of no pages.
    out = cache.attention(q, kv, 2, table[:, :5].contiguous(), offs, starts)
    held(out, step, 2, *f64.attention(step, q.cpu(), 2, f64.chain(step.new),
                                      missing=[(0, 2), (0, 3), (0, 5), (0, 6), (1, 0)]))
    out = cache.attention(q, kv, 2, table[:, :0].contiguous(), offs, starts)
    assert float(out.abs().max()) == 0.0


@pytest.mark.parametrize("offsets", [[3, 1, 5], [0, 6, 2], [-4, 2, 5], [9, 9, 9]])
def test_offsets_out_of_order_stay_in_bounds(ncm, cuda, offsets):
    step = f64.Step(15, [2, 3], [20, 30], 1, 64, 16, BF16)
    kv, table, _, starts = step.to(cuda)
    q = queries(step, 2, cuda)
    buf = torch.full((7, 128), 5.0, dtype=BF16, device=cuda)
    cache.attention(q, kv, 2, table, torch.tensor(offsets, dtype=torch.int32, device=cuda), starts,
                    out=buf[1:6])
    torch.cuda.synchronize()
    assert bool((buf[[0, 6]] == 5.0).all())


def test_rows_of_no_request_and_other_columns_stay(ncm, cuda):
    """Padded steps: rows behind the last request, requests of no rows; q and
    out as columns of wider buffers."""
    step = f64.Step(16, [1, 0, 2, 0], [30, 500, 7, 0], 2, 64, 16, I8, extra_rows=4)
    kv, table, offs, starts = step.to(cuda)
    wide = torch.randn(7, 512, generator=torch.Generator().manual_seed(2)).to(BF16).to(cuda)
    buf = torch.full((7, 400), 9.0, dtype=BF16, device=cuda)
    out = buf[:, 16:272]
    assert cache.attention(wide[:, 128:384], kv, 4, table, offs, starts, out=out) is out
    ref, mag = f64.attention(step, wide.cpu()[:, 128:384], 4, f64.chain(step.new))
    held(out, step, 4, ref, mag)
    rest = torch.ones(7, 400, dtype=torch.bool)
    rest[:3, 16:272] = False
    assert bool((buf.cpu()[rest] == 9.0).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_layers_in_one_buffer_and_a_slice_of_a_table(ncm, cuda, dtype):
    """K, V and scales as parts of wider buffers that hold NaN elsewhere, the
    page table as columns of a wider one."""
    step = f64.Step(23, [3, 1, 6], [200, 90, 0], 2, 64, 32, dtype)
    q = queries(step, 4, cuda)
    kv, table, offs, starts = step.to(cuda)
    ref = cache.attention(q, kv, 4, table, offs, starts)
    held(ref, step, 4, *f64.attention(step, q.cpu(), 4, f64.chain(step.new)))
    pages = kv.k.shape[0]
    byte = torch.full((pages, 3, 2, *kv.k.shape[1:]), 127, dtype=torch.uint8, device=cuda)
    wide = byte.view(dtype) if dtype != BF16 else torch.full(byte.shape, math.nan, dtype=BF16,
                                                              device=cuda)
    wide[:, 1, 0], wide[:, 1, 1] = kv.k, kv.v
    scales = (None, None)
    if dtype != BF16:
        sc = torch.full((pages, 2, 2, *kv.k_scale.shape[1:]), math.nan, device=cuda)
        sc[:, 1, 0], sc[:, 1, 1] = kv.k_scale, kv.v_scale
        scales = sc[:, 1, 0], sc[:, 1, 1]
    part = cache.KvCache(wide[:, 1, 0], wide[:, 1, 1], *scales)
    cols = torch.full((3, table.shape[1] + 5), 2**31 - 1, dtype=torch.int32, device=cuda)
    cols[:, 2:2 + table.shape[1]] = table
    out = cache.attention(q, part, 4, cols[:, 2:2 + table.shape[1]], offs, starts)
    assert torch.equal(out, ref)


def test_many_requests(ncm, cuda):
    """More requests than a workgroup has threads, most of them short."""
    rng = np.random.default_rng(3)
    n = 700
    new = [int(x) for x in rng.integers(0, 3, n)]
    before = [int(x) for x in rng.integers(0, 40, n)]
    before[n - 2], new[n - 2] = 900, 2
    step = f64.Step(17, new, before, 1, 64, 16, BF16)
    q, out = run(step, 2, cuda)
    held(out, step, 2, *f64.attention(step, q, 2, f64.chain(new)))


@pytest.mark.parametrize("dtype", DTYPES)
def test_long_and_ragged(ncm, cuda, dtype):
    """A long request split over many workgroups beside short ones, a tree."""
    new, before = [9, 1, 30], [9000, 3, 2500]
    step = f64.Step(18, new, before, 1, 64, 64, dtype)
    allowed = f64.tree(1, new)
    q, out = run(step, 4, cuda, allowed, 1)
    held(out, step, 4, *f64.attention(step, q, 4, allowed))


def test_same_bits_again_and_on_other_streams(ncm, cuda):
    """Equal calls give equal bits, two at once on two streams too."""
    step = f64.Step(19, [12, 1], [3000, 700], 2, 64, 16, FP8)
    kv, table, offs, starts = step.to(cuda)
    q = queries(step, 8, cuda)
    ref = cache.attention(q, kv, 8, table, offs, starts)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for k in range(6):
        with torch.cuda.stream(streams[k % 2]):
            outs.append(cache.attention(q, kv, 8, table, offs, starts))
    torch.cuda.synchronize()
    assert all(torch.equal(o, ref) for o in outs)


def test_capture(ncm, cuda):
    """Two captured steps, replayed with other lengths, beside eager calls."""
    step = f64.Step(20, [4, 4], [300, 50], 2, 64, 16, I8)
    kv, table, offs, starts = step.to(cuda)
    q = queries(step, 4, cuda)
    outs = [torch.zeros(8, 256, dtype=BF16, device=cuda) for _ in range(2)]
    mask = f64.bits(f64.tree(2, [4, 4]), 8, 1).to(cuda)
    cache.attention(q, kv, 4, table, offs, starts)
    torch.cuda.synchronize()
    graphs = []
    for out, m in zip(outs, (mask, None)):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            cache.attention(q, kv, 4, table, offs, starts, tree_mask=m, out=out)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for a, b in ((300, 50), (17, 0), (250, 31)):
        starts.copy_(torch.tensor([a, b]))
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for out, m in zip(outs, (mask, None)):
            assert torch.equal(out, cache.attention(q, kv, 4, table, offs, starts, tree_mask=m))


def test_refusals(ncm, cuda):
    step = f64.Step(21, [2], [5], 2, 64, 16, BF16)
    kv, table, offs, starts = step.to(cuda)
    q = queries(step, 4, cuda)
    with pytest.raises(NcmError):
        cache.attention(q, kv, 3, table, offs, starts)                   # 3 heads over 2
    with pytest.raises(NcmError):
        cache.attention(q, kv, 4, table, offs, starts, window=-1)
    with pytest.raises(NcmError):
        cache.attention(q[:, 1:129], kv, 2, table, offs, starts)         # alignment
    with pytest.raises(NcmError):
        cache.attention(q, kv, 4, table, offs, starts,                   # too small
                        workspace=torch.zeros(8, dtype=torch.uint8, device=cuda))
