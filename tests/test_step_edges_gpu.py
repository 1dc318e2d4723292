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
