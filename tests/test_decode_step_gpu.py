"""The operators that continue a sequence run together, as a decoder's step: a
chunked prefill into the cache, then drafted trees behind it, their logits
adjusted. Logits against the decoder's own prefill of every path, by the bound
that both are held to against exact arithmetic (3% of the largest logit each:
6% between them)."""
import numpy as np
import pytest
import torch

from ncmorph_amd import cache, decoder, kernels
from ncmorph_amd.context import Context
from tests import step_f64 as f64

pytestmark = pytest.mark.gpu

I32 = torch.int32


def step(spec, weights, inv, kvs, ids, positions, table, offsets, starts, mask=None, ctx=None):
    """Logits of a step's rows; every layer's cache gets their K and V."""
    hd, qh, kh = spec.head_dim, spec.q_heads, spec.kv_heads
    qw, kw, n = qh * hd, kh * hd, ids.numel()
    x = weights.embed[ids].float()
    for layer, kv in zip(weights.layers, kvs):
        y = kernels.rms_norm_rows(x, layer["input_norm"], spec.rms_eps, out_mode="bf16", ctx=ctx)
        qkv = torch.empty(n, spec.qkv_width, dtype=torch.bfloat16, device=x.device)
        kernels.linear_bf16(y, layer["qkv_weight"], out=qkv, out_mode="bf16", ctx=ctx)
        rot = qkv[:, :qw + kw]
        kernels.rope_positions(rot, positions, inv, qh + kh, hd, out=rot)
        cache.write(kv, qkv[:, qw:qw + kw], qkv[:, qw + kw:], table, offsets, starts)
        o = cache.attention(qkv[:, :qw], kv, qh, table, offsets, starts, tree_mask=mask,
                            window=spec.window, positions=positions)
        x = kernels.linear_bf16_residual(o, layer["o_weight"], x, ctx=ctx)
        y = kernels.rms_norm_rows(x, layer["post_attention_norm"], spec.rms_eps, out_mode="bf16",
                                  ctx=ctx)
        y = kernels.linear_bf16_swiglu(y, layer["gate_up_weight"], ctx=ctx)
        x = kernels.linear_bf16_residual(y, layer["down_weight"], x, ctx=ctx)
    y = kernels.rms_norm_rows(x, weights.final_norm, spec.rms_eps, out_mode="bf16", ctx=ctx)
    return kernels.linear_bf16(y, weights.embed if weights.lm_head is None else weights.lm_head,
                               out_mode="bf16_f32", ctx=ctx)


def ints(v, cuda):
    return torch.tensor(v, dtype=I32, device=cuda)


def tables(spec, n, cuda):
    return tuple(torch.from_numpy(t).to(cuda) for t in decoder.rope_tables(spec, n))


@pytest.mark.parametrize("hd,window", [(64, 0), (128, 0), (64, 24)])
def test_prefill_then_trees(ncm, cuda, hd, window):
    spec = decoder.DecoderSpec(hidden=256, intermediate=512, vocab=1000, q_heads=4, kv_heads=2,
                               head_dim=hd, layers=2, window=window)
    weights = decoder.random_weights(spec, cuda, seed=3)
    inv = torch.from_numpy(decoder.rope_inverse_frequencies(spec)).to(cuda)
    rng = np.random.default_rng(5)
    prompts = [rng.integers(0, spec.vocab, n) for n in (40, 17, 1)]
    drafts = [rng.integers(0, spec.vocab, n) for n in (7, 3, 12)]
    kvs = [cache.allocate(12, 2, 16, hd, torch.bfloat16, cuda) for _ in range(spec.layers)]
    table = ints([[7, 2, 9, 11], [0, 5, -1, -1], [3, -1, -1, -1]], cuda)

    def close(got, ref):
        assert float((got - ref).abs().max()) <= 0.06 * float(ref.abs().max())

    # Prompts in two chunks: all but their last tokens, then those.
    first = [p[:-1] for p in prompts]
    offs = np.cumsum([0] + [len(p) for p in first])
    step(spec, weights, inv, kvs, torch.from_numpy(np.concatenate(first)).to(cuda),
         ints(np.concatenate([np.arange(len(p)) for p in first]), cuda), table, ints(offs, cuda),
         ints([0, 0, 0], cuda))
    last = torch.tensor([int(p[-1]) for p in prompts], device=cuda)
    at = ints([len(p) - 1 for p in prompts], cuda)
    got = step(spec, weights, inv, kvs, last, at, table, ints([0, 1, 2, 3], cuda), at)
    for r, p in enumerate(prompts):
        ref = decoder.forward(spec, weights, p[None], *tables(spec, len(p), cuda))
        close(got[r], ref[-1])
    # Trees behind them: every row as the last token of its own path.
    seen = f64.tree(6, [len(d) for d in drafts])
    rows = sum(len(d) for d in drafts)
    offsets = ints(np.cumsum([0] + [len(d) for d in drafts]), cuda)
    starts = ints([len(p) for p in prompts], cuda)
    pos = torch.cat([s.sum(1) - 1 + len(p) for s, p in zip(seen, prompts)]).to(I32).to(cuda)
    mask = f64.bits(seen, rows, 1).to(cuda)
    ids = torch.from_numpy(np.concatenate(drafts)).to(cuda)
    got = step(spec, weights, inv, kvs, ids, pos, table, offsets, starts, mask)
    i = 0
    for p, d, s in zip(prompts, drafts, seen):
        for t in range(len(d)):
            path = np.concatenate([p, d[np.flatnonzero(s[t].numpy())]])
            if not window:
                ref = decoder.forward(spec, weights, path[None], *tables(spec, len(path), cuda))
                close(got[i], ref[-1])
            i += 1
    # Penalties over prompt and path.
    width = max(len(p) for p in prompts)
    history = torch.zeros(3, width, dtype=I32)
    for r, p in enumerate(prompts):
        history[r, :len(p)] = torch.from_numpy(p)
    lens = torch.tensor([len(p) for p in prompts], dtype=I32)
    y = kernels.adjust_logits(got, history=history.to(cuda), prompt_lens=(lens - 1).to(cuda),
                              history_lens=lens.to(cuda),
                              repetition=torch.full((3,), 1.3, device=cuda),
                              frequency=torch.full((3,), 0.5, device=cuda), offsets=offsets,
                              draft_tokens=ids.int(), tree_mask=mask)
    i = 0
    for p, d, s in zip(prompts, drafts, seen):
        for t in range(len(d)):
            path = d[np.flatnonzero(s[t].numpy())]
            made = np.bincount(np.concatenate([p[-1:], path]), minlength=1000)
            was = (made > 0) | (np.bincount(p, minlength=1000) > 0)
            x = got[i].double().cpu().numpy()
            ref = np.where(was, np.where(x > 0, x / np.float64(np.float32(1.3)),
                                         x * np.float64(np.float32(1.3))), x) - 0.5 * made
            assert np.allclose(y[i].double().cpu().numpy(), ref, rtol=2.0 ** -21, atol=2.0 ** -21)
            i += 1


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn, torch.int8])
def test_captured_steps(ncm, cuda, dtype):
    """One captured step, replayed token after token, gives the eager steps'
    logits and cache bit for bit, with eager work between the replays."""
    spec = decoder.DecoderSpec(hidden=256, intermediate=512, vocab=1000, q_heads=4, kv_heads=2,
                               head_dim=64, layers=2)
    weights = decoder.random_weights(spec, cuda, seed=3)
    inv = torch.from_numpy(decoder.rope_inverse_frequencies(spec)).to(cuda)
    table = ints([[3, 1], [0, 2]], cuda)
    offs = ints([0, 1, 2], cuda)

    def fresh():
        return [cache.allocate(4, 2, 16, 64, dtype, cuda) for _ in range(spec.layers)]

    kvs, eager = fresh(), fresh()
    ids = torch.zeros(2, dtype=torch.int64, device=cuda)
    starts = torch.zeros(2, dtype=I32, device=cuda)
    ctx = Context(0)
    step(spec, weights, inv, fresh(), ids, starts, table, offs, starts, ctx=ctx)  # warm
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits = step(spec, weights, inv, kvs, ids, starts, table, offs, starts, ctx=ctx)
    for t in range(20):
        ids.copy_(torch.tensor([17 * t % 1000, 31 * t % 1000]))
        starts.copy_(torch.tensor([t, t]))
        graph.replay()
        ref = step(spec, weights, inv, eager, ids, starts, table, offs, starts)
        torch.cuda.synchronize()
        assert torch.equal(logits, ref), t
    for a, b in zip(kvs, eager):
        assert torch.equal(a.k.view(torch.uint8), b.k.view(torch.uint8))
        assert torch.equal(a.v.view(torch.uint8), b.v.view(torch.uint8))
