"""Penalties, biases and masks on logits against 64-bit arithmetic: one
rounding for the penalty's quotient or product, one each for the two
subtractions, the frequency's product, the bias's sum and its addition, each
2^-24 of a value no larger than |x| rep + freq count + pres + sum |bias|;
bfloat16 outputs add 2^-8 of the result."""
import math

import numpy as np
import pytest
import torch

from ncmorph_amd import kernels
from ncmorph_amd._lib import NcmError
from tests import step_f64 as f64

pytestmark = pytest.mark.gpu

I32 = torch.int32


def rules(seed, requests, rows, vocab, width, nb, mask=True):
    g = torch.Generator().manual_seed(seed)
    h = (torch.rand(requests, width, generator=g) ** 3 * (vocab + 6)).to(I32) - 3
    lens = torch.randint(0, width + 2, (requests,), generator=g, dtype=I32)
    r = dict(history=h, history_lens=lens, prompt_lens=lens // 2 - 1,
             repetition=0.7 + torch.rand(requests, generator=g),
             frequency=torch.rand(requests, generator=g) - 0.3,
             presence=torch.rand(requests, generator=g) - 0.3)
    if nb:   # ids from a few tokens, so that they repeat, some outside
        r["bias_ids"] = torch.randint(-2, min(vocab, 3 * nb) + 2, (requests, nb), generator=g,
                                      dtype=I32)
        r["bias_values"] = torch.randn(requests, nb, generator=g) * 5
    if mask:
        r["allowed"] = torch.randint(-2**31, 2**31, (rows, (vocab + 31) // 32), generator=g).to(I32)
    return r


def reference(x, r, requests, offsets=None, draft=None, seen_rows=None):
    """(values, tolerances without the output's rounding) in 64 bits; rows of no
    request NaN."""
    rows, v = x.shape
    offs = list(range(rows + 1)) if offsets is None else offsets
    out = torch.full((rows, v), math.nan, dtype=torch.float64)
    tol = torch.zeros(rows, v, dtype=torch.float64)
    for q in range(requests):
        count0, old = np.zeros(v), np.zeros(v, bool)
        if r.get("history") is not None:
            h, width = r["history"][q].numpy(), r["history"].shape[1]
            p = 0 if r.get("prompt_lens") is None else min(max(int(r["prompt_lens"][q]), 0), width)
            n = width if r.get("history_lens") is None else min(max(int(r["history_lens"][q]), 0),
                                                                width)
            for t in h[:p]:
                if 0 <= t < v:
                    old[t] = True
            for t in h[p:n]:
                if 0 <= t < v:
                    count0[t] += 1
        bias, mag = np.zeros(v), np.zeros(v)
        for t, b in zip(*(([], []) if r.get("bias_ids") is None else
                          (r["bias_ids"][q].tolist(), r["bias_values"][q].tolist()))):
            if 0 <= t < v:
                bias[t] += b
                mag[t] += abs(b)
        get = lambda n, d: d if r.get(n) is None else float(r[n][q])  # noqa: E731
        rep, freq, pres = get("repetition", 1.0), get("frequency", 0.0), get("presence", 0.0)
        for i in range(offs[q], offs[q + 1]):
            count = count0.copy()
            if draft is not None:
                for j in range(offs[q + 1] - offs[q]):
                    t = int(draft[offs[q] + j])
                    if bool(seen_rows[q][i - offs[q]][j]) and 0 <= t < v:
                        count[t] += 1
            y = x[i].double().numpy()
            was = old | (count > 0)
            with np.errstate(invalid="ignore"):
                y = np.where(was, np.where(y > 0, y / rep, y * rep), y)
                y = y - freq * count - pres * (count > 0) + bias
                size = (np.abs(x[i].double().numpy()) * max(rep, 1 / rep, 1.0)
                        + abs(freq) * count + abs(pres) + mag)
            if r.get("allowed") is not None:
                w = r["allowed"][i].numpy().view(np.uint32)
                ok = (w[np.arange(v) // 32] >> (np.arange(v) % 32).astype(np.uint32)) & 1
                y = np.where(ok == 1, y, -math.inf)
            out[i], tol[i] = torch.from_numpy(y), torch.from_numpy(size * 8 * 2.0 ** -24)
    return out, tol


def held(y, ref, tol):
    y = y.cpu()
    if y.dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * ref.abs()
    fine = torch.isfinite(ref)
    assert torch.equal(torch.isnan(y), torch.isnan(ref))
    both = ~fine & ~torch.isnan(ref)
    assert torch.equal(y.double()[both], ref[both])
    err = (y.double() - ref).abs()[fine]
    assert bool((err <= tol[fine]).all()), float((err / (tol[fine] + 1e-300)).max())


def to(r, cuda):
    return {k: None if t is None else t.to(cuda) for k, t in r.items()}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,width,nb", [
    (1, 1, 1, 1), (1, 5, 3, 2), (3, 33, 40, 7), (2, 2048, 600, 0), (2, 8195, 2000, 300),
    (5, 50257, 300, 20), (70, 1000, 64, 9), (1, 151936, 5000, 300), (128, 66003, 300, 9)])
def test_rules(ncm, cuda, rows, vocab, width, nb, dtype):
    x = (torch.randn(rows, vocab, generator=torch.Generator().manual_seed(1)) * 4).to(dtype)
    r = rules(2, rows, rows, vocab, width, nb)
    y = kernels.adjust_logits(x.to(cuda), **to(r, cuda))
    held(y, *reference(x, r, rows))
    # In place, the same bits; the same call again, the same bits.
    z = x.to(cuda)
    assert kernels.adjust_logits(z, out=z, **to(r, cuda)) is z
    as_int = torch.int32 if dtype == torch.float32 else torch.int16
    assert torch.equal(z.view(as_int), y.view(as_int))


@pytest.mark.parametrize("left", ["history", "bias", "mask", "penalties", "none"])
def test_each_rule_alone(ncm, cuda, left):
    x = torch.randn(3, 4099, generator=torch.Generator().manual_seed(1)) * 4
    r = rules(3, 3, 3, 4099, 500, 20)
    keep = {"history": ("history", "repetition", "frequency"), "bias": ("bias_ids", "bias_values"),
            "mask": ("allowed",), "penalties": ("repetition", "presence"), "none": ()}[left]
    r = {k: v for k, v in r.items() if k in keep}
    y = kernels.adjust_logits(x.to(cuda), **to(r, cuda))
    held(y, *reference(x, r, 3))


@pytest.mark.parametrize("words", [0, 1, 2])
def test_drafted_trees(ncm, cuda, words):
    """Rows of requests, their paths counted (words 0: chains); requests of no
    rows, rows of no request left as they were."""
    new, vocab = [4, 0, 1, 70 if words != 1 else 40], 700
    rows = sum(new) + 2
    offs = [0] + list(np.cumsum(new))
    seen = f64.tree(5, new) if words else f64.chain(new)
    r = rules(6, 4, rows, vocab, 60, 12)
    draft = torch.randint(-1, 30, (rows,), generator=torch.Generator().manual_seed(8)).to(I32)
    x = torch.randn(rows, vocab, generator=torch.Generator().manual_seed(1)) * 4
    out = torch.full((rows, vocab + 5), 7.0, device=cuda)
    y = kernels.adjust_logits(
        x.to(cuda), offsets=torch.tensor(offs, dtype=I32, device=cuda), draft_tokens=draft.to(cuda),
        tree_mask=f64.bits(seen, rows, words).to(cuda) if words else None, out=out[:, 2:vocab + 2],
        **to(r, cuda))
    ref, tol = reference(x, r, 4, offs, draft, seen)
    held(y[:-2], ref[:-2], tol[:-2])
    assert bool((out[-2:] == 7.0).all()) and bool((out[:, :2] == 7.0).all())
    assert bool((out[:, vocab + 2:] == 7.0).all())


@pytest.mark.parametrize("offsets", [[3, 1, 5], [0, 6, 2], [-4, 2, 5], [9, 9, 9]])
def test_offsets_out_of_order_stay_in_bounds(ncm, cuda, offsets):
    r = rules(6, 2, 5, 100, 20, 3)
    buf = torch.full((7, 100), 7.0, device=cuda)
    kernels.adjust_logits(torch.zeros(5, 100, device=cuda), out=buf[1:6], **to(r, cuda),
                          offsets=torch.tensor(offsets, dtype=I32, device=cuda),
                          draft_tokens=torch.zeros(5, dtype=I32, device=cuda),
                          tree_mask=torch.full((5, 1), -1, device=cuda))
    torch.cuda.synchronize()
    assert bool((buf[[0, 6]] == 7.0).all())


def test_many_requests(ncm, cuda):
    """More requests than a workgroup has threads."""
    new = [int(t) for t in np.random.default_rng(1).integers(0, 3, 600)]
    rows, offs = sum(new), [0] + list(np.cumsum(new))
    r = rules(9, 600, rows, 65, 10, 2)
    x = torch.randn(rows, 65, generator=torch.Generator().manual_seed(1))
    y = kernels.adjust_logits(x.to(cuda), offsets=torch.tensor(offs, dtype=I32, device=cuda),
                              **to(r, cuda))
    held(y, *reference(x, r, 600, offs))


def test_values_that_are_not_finite(ncm, cuda):
    """NaN and infinities go through the arithmetic; a mask wins over them, and
    a row whose mask allows nothing is all -infinity."""
    vals = [math.nan, math.inf, -math.inf, 0.0, -0.0, 3.4e38, -3.4e38, 1e-40]
    x = torch.tensor([vals * 4] * 3)
    r = dict(history=torch.arange(16, dtype=I32).repeat(3, 1), repetition=torch.full((3,), 1.5),
             frequency=torch.full((3,), 0.5), presence=torch.full((3,), 0.25),
             allowed=torch.tensor([[-1], [0x0F0F0F0F], [0]], dtype=I32))
    y = kernels.adjust_logits(x.to(cuda), **to(r, cuda))
    ref, tol = reference(x, r, 3)
    big = ref.abs() > 3.4028235677973366e38
    ref[big] = torch.sign(ref[big]) * math.inf       # float32's range
    held(y, ref, tol)
    assert bool((y[2] == -math.inf).all())


def test_strides(ncm, cuda):
    """Row strides, alignments that differ between in and out, empty sizes."""
    g = torch.Generator().manual_seed(1)
    for a, b in ((0, 0), (1, 1), (1, 2), (3, 0)):
        buf = torch.randn(4, 3001, generator=g).to(cuda)
        x = buf[:, a:a + 2990]
        r = rules(4, 4, 4, 2990, 100, 9)
        out = torch.full((4, 3003), 7.0, device=cuda)
        y = kernels.adjust_logits(x, out=out[:, b:b + 2990], **to(r, cuda))
        held(y, *reference(x.cpu(), r, 4))
        assert bool((out[:, :b] == 7.0).all()) and bool((out[:, b + 2990:] == 7.0).all())
    assert kernels.adjust_logits(torch.zeros(0, 9, device=cuda)).shape == (0, 9)
    assert kernels.adjust_logits(torch.zeros(9, 0, device=cuda)).shape == (9, 0)


def test_capture(ncm, cuda):
    x = torch.randn(3, 5000, device=cuda)
    r = to(rules(5, 3, 3, 5000, 200, 9), cuda)
    y = torch.empty_like(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kernels.adjust_logits(x, out=y, **r)
    for k in range(3):
        x.copy_(torch.randn(3, 5000, device=cuda))
        r["history_lens"].fill_(50 * k)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, kernels.adjust_logits(x, **r))


def test_refusals(ncm, cuda):
    x = torch.zeros(2, 50, device=cuda)
    z = lambda *s, d=I32: torch.zeros(s, dtype=d, device=cuda)  # noqa: E731
    f = torch.float32
    for kw in (dict(history=z(3, 4)), dict(prompt_lens=z(2)), dict(repetition=z(3, d=f)),
               dict(bias_ids=z(2, 3)), dict(bias_ids=z(2, 3), bias_values=z(2, 4, d=f)),
               dict(allowed=z(2, 1)), dict(allowed=z(1, 2)), dict(draft_tokens=z(2)),
               dict(tree_mask=z(2, 1, d=torch.int64)), dict(out=z(2, 49, d=f)),
               dict(out=z(2, 50, d=torch.bfloat16)), dict(offsets=z(0)), dict(frequency=z(2))):
        with pytest.raises(NcmError):
            kernels.adjust_logits(x, **kw)
    with pytest.raises(NcmError):
        kernels.adjust_logits(x.half())
