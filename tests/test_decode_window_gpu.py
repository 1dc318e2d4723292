"""Windowed attention behind drafted trees: the step's logits against the
decoder's own windowed prefill of every path. A path is shorter than the window,
so all of its drafted tokens are in it, and a row's window over the tokens before
ends at its position, its depth in the tree; both are what the prefill does. By
the bound of the step without a window (3% of the largest logit each side)."""
import numpy as np
import pytest
import torch

from ncmorph_amd import cache, decoder
from tests import step_f64 as f64
from tests.test_decode_step_gpu import I32, ints, step, tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd,window", [(64, 24), (128, 16)])
def test_trees_under_a_window(ncm, cuda, hd, window):
    spec = decoder.DecoderSpec(hidden=256, intermediate=512, vocab=1000, q_heads=4, kv_heads=2,
                               head_dim=hd, layers=2, window=window)
    weights = decoder.random_weights(spec, cuda, seed=3)
    inv = torch.from_numpy(decoder.rope_inverse_frequencies(spec)).to(cuda)
    rng = np.random.default_rng(7)
    prompts = [rng.integers(0, spec.vocab, n) for n in (60, 17, 30)]
    drafts = [rng.integers(0, spec.vocab, n) for n in (9, 3, 12)]
    kvs = [cache.allocate(16, 2, 16, hd, torch.bfloat16, cuda) for _ in range(spec.layers)]
    table = ints([[7, 2, 9, 11, 15], [0, 5, -1, -1, -1], [3, 12, 1, -1, -1]], cuda)
    step(spec, weights, inv, kvs, torch.from_numpy(np.concatenate(prompts)).to(cuda),
         ints(np.concatenate([np.arange(len(p)) for p in prompts]), cuda), table,
         ints(np.cumsum([0] + [len(p) for p in prompts]), cuda), ints([0, 0, 0], cuda))
    seen = f64.tree(6, [len(d) for d in drafts])
    pos = torch.cat([s.sum(1) - 1 + len(p) for s, p in zip(seen, prompts)]).to(I32).to(cuda)
    got = step(spec, weights, inv, kvs, torch.from_numpy(np.concatenate(drafts)).to(cuda), pos,
               table, ints(np.cumsum([0] + [len(d) for d in drafts]), cuda),
               ints([len(p) for p in prompts], cuda),
               f64.bits(seen, sum(len(d) for d in drafts), 1).to(cuda))
    i = 0
    for p, d, s in zip(prompts, drafts, seen):
        for t in range(len(d)):
            path = np.concatenate([p, d[np.flatnonzero(s[t].numpy())]])
            ref = decoder.forward(spec, weights, path[None], *tables(spec, len(path), cuda))[-1]
            assert float((got[i] - ref).abs().max()) <= 0.06 * float(ref.abs().max()), (i, t)
            i += 1
