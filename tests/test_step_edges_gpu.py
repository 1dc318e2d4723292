"""Calls at the edges of what the operators that continue a sequence accept."""
import pytest
import torch

from ncmorph_amd import cache, kernels
from tests import step_f64 as f64
from tests.step_f64 import BF16, FP8, I8

pytestmark = pytest.mark.gpu

I32 = torch.int32


@pytest.mark.parametrize("dtype", [BF16, FP8, I8])
@pytest.mark.parametrize("before", [0, 40])
def test_a_tree_mask_of_no_words(ncm, cuda, dtype, before):
    """No new token is seen: the tokens before alone, or nothing."""
    step = f64.Step(3, [3, 2], [before, before], 1, 64, 16, dtype)
    kv, table, offs, starts = step.to(cuda)
    q = torch.randn(5, 128, generator=torch.Generator().manual_seed(2)).to(BF16).to(cuda)
    mask = torch.zeros(5, 0, dtype=torch.int64, device=cuda)
    out = cache.attention(q, kv, 2, table, offs, starts, tree_mask=mask)
    none = [torch.zeros(n, n).bool() for n in step.new]
    ref, mag = f64.attention(step, q.cpu(), 2, none)
    err = (out.cpu().double().view(5, 2, 64) - ref).abs()
    assert bool((err <= f64.attention_bound(ref, mag)).all())
    one = torch.zeros(5, 1, dtype=torch.int64, device=cuda)
    assert torch.equal(out, cache.attention(q, kv, 2, table, offs, starts, tree_mask=one))
    # A window holds for the tokens before alone.
    out = cache.attention(q, kv, 2, table, offs, starts, tree_mask=mask, window=7)
    assert torch.equal(out, cache.attention(q, kv, 2, table, offs, starts, tree_mask=one,
                                            window=7))


def test_a_tree_mask_of_no_words_counts_no_drafts(ncm, cuda):
    x = torch.randn(5, 300, device=cuda)
    kw = dict(offsets=torch.tensor([0, 3, 5], dtype=I32, device=cuda),
              draft_tokens=torch.arange(5, dtype=I32, device=cuda) % 2,
              frequency=torch.ones(2, device=cuda), presence=torch.ones(2, device=cuda))
    y = kernels.adjust_logits(x, tree_mask=torch.zeros(5, 0, dtype=torch.int64, device=cuda), **kw)
    assert torch.equal(y, x)


@pytest.mark.parametrize("dtype", [BF16, FP8, I8])
@pytest.mark.parametrize("form", ["chain", "tree", "positions"])
def test_windows_behind_a_short_table(ncm, cuda, dtype, form):
    """The table ends before the requests' own rows: their windows still end at
    their positions, not at the table's end."""
    step = f64.Step(9, [2, 3, 1], [100, 70, 300], 1, 64, 16, dtype)
    kv, table, offs, starts = step.to(cuda)
    q = torch.randn(6, 128, generator=torch.Generator().manual_seed(2)).to(BF16).to(cuda)
    allowed = f64.chain(step.new) if form == "chain" else f64.tree(2, step.new)
    mask = None if form == "chain" else f64.bits(allowed, 6, 1).to(cuda)
    pos = None
    if form == "positions":
        pos = torch.tensor([100, 103, 70, -1, 75, 280], dtype=I32)
    missing = [(r, p) for r in range(3) for p in range(4, 30)]
    for window in (1, 50, 90, 260):
        out = cache.attention(q, kv, 2, table[:, :4].contiguous(), offs, starts, tree_mask=mask,
                              window=window, positions=None if pos is None else pos.to(cuda))
        ref, mag = f64.attention(step, q.cpu(), 2, allowed, window=window, positions=pos,
                                 missing=missing, chained=form == "chain")
        err = (out.cpu().double().view(6, 2, 64) - ref).abs()
        assert bool((err <= f64.attention_bound(ref, mag)).all()), window


def equal_keys(seed, new, before, hd, dtype, key):
    """A step whose K hold `key` in every place; an equal score for all tokens."""
    step = f64.Step(seed, new, before, 1, hd, 16, dtype)
    for x in step.tokens[0]:
        x.fill_(key)
    codes, sc = f64.quantise(torch.full((1, hd), key).to(BF16), dtype)
    if dtype == BF16:
        step.pages[0][:] = codes[0]
    else:
        step.pages[0].view(torch.uint8)[:] = codes[0].view(torch.uint8)
        step.scales[0].fill_(float(sc[0]))
    return step


def means(out, step, hd):
    """Equal scores: every row is the mean of the V that it sees."""
    out = out.cpu().double().view(-1, 2, hd)
    V, i = step.cached(1), 0
    for r, (n, c) in enumerate(zip(step.new, step.before)):
        for j in range(n):
            v = V[r][:c + j + 1, 0]
            ref, mag = v.mean(0), v.abs().mean(0)
            assert bool(((out[i] - ref).abs() <= f64.attention_bound(ref, mag)).all()), (r, j)
            i += 1


@pytest.mark.parametrize("dtype", [BF16, FP8, I8])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("key", [2.0 ** 5, -2.0 ** 15, 2.0 ** 30, -2.0 ** 50, 2.0 ** 60])
def test_scores_of_any_size(ncm, cuda, dtype, hd, key):
    """Scores of 2^28 to 2^84, of both signs, the same bits for every token; of
    mantissas whose products with the scale are rounded."""
    step = equal_keys(5, [2, 1, 30], [0, 300, 2000], hd, dtype, 1.2890625 * key)
    kv, table, offs, starts = step.to(cuda)
    q = torch.full((33, 2 * hd), 1.5703125 * 2.0 ** 20, dtype=BF16, device=cuda)
    means(cache.attention(q, kv, 2, table, offs, starts), step, hd)


@pytest.mark.parametrize("far", [-2.0 ** 40, -2.0 ** 70, -2.0 ** 100])
def test_far_scores_beside_moderate_ones(ncm, cuda, far):
    """Tokens far below the others count for nothing, whole tiles of them too."""
    step = f64.Step(6, [1], [900], 1, 64, 16, BF16)
    step.tokens[0][0][50:] = 1.2890625 * far
    for t in range(50, 901):
        step.pages[0][int(step.table[0, t // 16]), 0, t % 16] = 1.2890625 * far
    kv, table, offs, starts = step.to(cuda)
    q = torch.full((1, 64), 1.5703125, dtype=BF16, device=cuda)
    out = cache.attention(q, kv, 1, table, offs, starts).cpu().double().view(1, 1, 64)
    ref, mag = f64.attention(step, q.cpu(), 1, f64.chain([1]))
    assert bool(((out - ref).abs() <= f64.attention_bound(ref, mag)).all())


@pytest.mark.parametrize("dtype", [BF16, FP8, I8])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("key", [-2.0 ** 42, -2.0 ** 50, -2.0 ** 57])
def test_scores_far_below_zero(ncm, cuda, dtype, hd, key):
    """All of a row's scores below -1e30, down to where 128 products of about
    2^118 still have a sum in fp32's range."""
    step = equal_keys(7, [2, 1, 30], [0, 300, 2000], hd, dtype, key)
    kv, table, offs, starts = step.to(cuda)
    q = torch.full((33, 2 * hd), 1.5703125 * 2.0 ** 60, dtype=BF16, device=cuda)
    means(cache.attention(q, kv, 2, table, offs, starts), step, hd)


def test_one_row_in_place_under_two_strides(ncm, cuda):
    """A single row has no stride: two views of it may name different ones."""
    buf = torch.randn(2, 200, generator=torch.Generator().manual_seed(2)).to(cuda)
    x, y = buf[:1, :128], buf.view(-1)[:128].view(1, 128)
    assert x.stride(0) != y.stride(0)
    pos = torch.tensor([1234], dtype=I32, device=cuda)
    inv = torch.rand(32, device=cuda)
    ref = kernels.rope_positions(x, pos, inv, 2, 64)
    assert kernels.rope_positions(x, pos, inv, 2, 64, out=y) is y
    assert torch.equal(x, ref)
    bias = dict(bias_ids=torch.tensor([[3, 90]], dtype=I32, device=cuda),
                bias_values=torch.tensor([[1.0, -2.0]], device=cuda))
    ref = kernels.adjust_logits(x, **bias)
    assert kernels.adjust_logits(x, out=y, **bias) is y
    assert torch.equal(x, ref)


@pytest.mark.parametrize("new,before", [([1, 1], [3000, 20]), ([70, 3], [100, 900])])
def test_attention_into_its_queries(ncm, cuda, new, before):
    """A unit's queries are read by the units that write their places alone, the
    parts of one that is cut before its join."""
    step = f64.Step(7, new, before, 2, 64, 16, BF16)
    kv, table, offs, starts = step.to(cuda)
    buf = torch.randn(step.rows, 400, generator=torch.Generator().manual_seed(2)).to(BF16).to(cuda)
    q = buf[:, 8:264]
    ref = cache.attention(q, kv, 4, table, offs, starts)
    was = buf.clone()
    assert cache.attention(q, kv, 4, table, offs, starts, out=q) is q
    assert torch.equal(q, ref)
    assert torch.equal(buf[:, :8], was[:, :8]) and torch.equal(buf[:, 264:], was[:, 264:])


def test_rows_before_the_first_request(ncm, cuda):
    """offsets that begin past 0: the rows ahead are no request's."""
    step = f64.Step(11, [3, 2], [40, 7], 2, 64, 16, BF16, extra_rows=4)
    kv, table, offs, starts = step.to(cuda)
    offs = offs + 3
    q = torch.randn(9, 256, generator=torch.Generator().manual_seed(2)).to(BF16).to(cuda)
    out = torch.full((9, 256), 5.0, dtype=BF16, device=cuda)
    cache.attention(q, kv, 4, table, offs, starts, out=out)
    ref, mag = f64.attention(step, q.cpu()[3:], 4, f64.chain(step.new))
    err = (out.cpu().double()[3:8].view(5, 4, 64) - ref[:5]).abs()
    assert bool((err <= f64.attention_bound(ref[:5], mag[:5])).all())
    k, v = (torch.full((9, 128), 5.0, dtype=BF16, device=cuda) for _ in range(2))
    cache.read(kv, table, offs, starts, 9, out=(k, v))
    for w, t in enumerate((k, v)):
        want = torch.cat([step.tokens[w][0][40:], step.tokens[w][1][7:]]).reshape(5, 128)
        assert torch.equal(t.cpu()[3:8], want)
    fresh = cache.allocate(kv.k.shape[0], 2, 16, 64, BF16, cuda)
    cache.write(fresh, k, v, table, offs, starts)
    x = torch.randn(9, 77, device=cuda)
    y = torch.full((9, 77), 5.0, device=cuda)
    one = torch.ones(2, device=cuda)
    kernels.adjust_logits(x, offsets=offs, out=y, presence=one,
                          history=torch.tensor([[3], [4]], dtype=I32, device=cuda))
    z = x.clone()
    z[3:6, 3] -= 1
    z[6:8, 4] -= 1
    assert torch.equal(y[3:8], z[3:8])
    for t in (out, k, v, y):
        assert bool((t[[0, 1, 2, 8]] == 5.0).all())
    k2, _ = cache.read(fresh, table, offs, starts, 9)
    assert torch.equal(k2[3:8], k[3:8])
    assert int((fresh.k != 0).any(-1).sum()) == 10     # five tokens of two heads


@pytest.mark.parametrize("dtype", [BF16, FP8, I8])
@pytest.mark.parametrize("scale", [0.0, 1e-45, -1e-38])
@pytest.mark.parametrize("key", [1.0, 2.0 ** 57, -2.0 ** 57])
def test_scales_of_nothing(ncm, cuda, dtype, scale, key):
    """Scores of 0 or next to it, also of products next to fp32's end."""
    step = equal_keys(8, [2, 1, 30], [0, 300, 2000], 64, dtype, 1.2890625 * key)
    kv, table, offs, starts = step.to(cuda)
    q = torch.full((33, 128), 1.5703125 * max(abs(key) * 8, 1.0), dtype=BF16, device=cuda)
    means(cache.attention(q, kv, 2, table, offs, starts, scale=scale), step, 64)
