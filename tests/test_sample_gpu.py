"""Token sampling (kernels.sample) against its definition in exact arithmetic:
the weights' integers and their sums as Python and numpy make them. Tokens are
equal; a probability is one quotient, rounded to float32 (2^-24) from 64-bit
values whose weights are good to one unit of 2^-43."""
import math

import numpy as np
import pytest
import torch

from ncmorph_amd import kernels

pytestmark = pytest.mark.gpu

F32, BF16, I32 = torch.float32, torch.bfloat16, torch.int32
ONE = 1 << 43


def plain(x, u, t=1.0, k=0, p=1.0, m=0.0):
    """(token, probability) of one row of float32 values."""
    x = np.array(x, np.float32)
    x = np.where(np.isnan(x), -np.inf, np.minimum(x, np.finfo(np.float32).max)).astype(np.float32)
    ids = np.flatnonzero(x > -np.inf)
    if not len(ids):
        return -1, 0.0
    ids = ids[np.argsort(-x[ids].astype(np.float64), kind="stable")]
    if not t > 0:
        return int(ids[0]), 1.0
    t = max(float(np.float32(t)), 2.0 ** -96)
    v = x[ids].astype(np.float64)
    with np.errstate(over="ignore", under="ignore"):
        w = np.rint(np.exp((v - v[0]) / t) * ONE).astype(np.uint64)
    if k > 0:
        w = w[:k]
    c = np.cumsum(w, dtype=np.uint64)
    kept = len(w)
    p = float(np.float32(p))
    if p < 1:
        need = max(math.ceil(_exact(max(p, 0.0)) * int(c[-1])), 1)
        kept = int(np.searchsorted(c, np.uint64(need))) + 1
    m = float(np.float32(m))
    if m > 0:
        kept = min(kept, int((w >= max(math.ceil(_exact(min(m, 1.0)) * ONE), 1)).sum()))
    total = int(c[kept - 1])
    u = min(max(u, 0.0), 1 - 2.0 ** -53) if u == u else 0.0
    at = int(np.searchsorted(c, np.uint64(math.floor(_exact(u) * total) + 1)))
    return int(ids[at]), int(w[at]) / total


def _exact(f):
    from fractions import Fraction

    return Fraction(f)


def on(v, dtype, cuda):
    return None if v is None else torch.as_tensor(np.asarray(v)).to(dtype).to(cuda)


def run(cuda, x, u, t=None, k=None, p=None, m=None, offsets=None, wide=False):
    x = x.to(cuda)
    return kernels.sample(x, on(u, torch.float64 if wide else F32, cuda), on(t, F32, cuda),
                          on(k, I32, cuda), on(p, F32, cuda), on(m, F32, cuda),
                          on(offsets, I32, cuda), probabilities=True)


def compare(cuda, x, u, t=None, k=None, p=None, m=None, request=None, wide=False, **kw):
    got, share = run(cuda, x, u, t, k, p, m, wide=wide, **kw)
    got, share = got.tolist(), share.tolist()
    u = np.asarray(u, np.float64 if wide else np.float32).astype(np.float64)
    rows = x.float().numpy()
    for i in range(len(rows)):
        r = i if request is None else request[i]
        if r is None:
            continue
        want, chance = plain(rows[i], u[i], 1.0 if t is None else t[r], 0 if k is None else k[r],
                             1.0 if p is None else p[r], 0.0 if m is None else m[r])
        assert got[i] == want, (i, got[i], want)
        assert abs(share[i] - chance) <= 2.0 ** -24 * chance + 2.0 ** -42, (i, share[i], chance)


def rules(g, n):
    return dict(t=np.where(g.random(n) < 0.1, 0, g.uniform(0.3, 2.0, n)).astype(np.float32),
                k=np.where(g.random(n) < 0.4, 0, g.integers(1, 300, n)),
                p=np.where(g.random(n) < 0.4, 1, g.uniform(0.05, 1, n)).astype(np.float32),
                m=np.where(g.random(n) < 0.5, 0, g.uniform(0, 0.3, n)).astype(np.float32))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (5, 2), (9, 7), (33, 63), (64, 1000), (300, 4097),
                                        (1, 49152), (3, 50257), (40, 50257), (16, 151936),
                                        (2, 1 << 20)])
def test_rules(cuda, dtype, rows, vocab):
    g = np.random.default_rng(rows + vocab)
    x = torch.from_numpy((g.uniform(0.5, 5, (rows, 1)) * g.standard_normal((rows, vocab)))
                         .astype(np.float32)).to(dtype)
    x[torch.from_numpy(g.random((rows, vocab)) < 0.2)] = -math.inf
    compare(cuda, x, g.random(rows), **rules(g, rows))


@pytest.mark.parametrize("vocab", [5, 1000, 40000])
def test_each_rule_alone(cuda, vocab):
    g = np.random.default_rng(vocab)
    x = torch.from_numpy((3 * g.standard_normal((24, vocab))).astype(np.float32))
    u = g.random(24)
    compare(cuda, x, u)
    compare(cuda, x, u, t=g.uniform(0.05, 10, 24))
    compare(cuda, x, u, k=g.integers(1, vocab + 5, 24))
    compare(cuda, x, u, p=g.uniform(0, 1, 24))
    compare(cuda, x, u, m=g.uniform(0, 1, 24))
    compare(cuda, x, u, wide=True)


@pytest.mark.parametrize("vocab", [4, 1000, 100000])
@pytest.mark.parametrize("values", [1, 3])
def test_ties(cuda, vocab, values):
    """Few different logits: ids decide, at cuts and at draws on borders."""
    g = np.random.default_rng(values)
    x = torch.from_numpy(g.integers(0, values, (32, vocab)).astype(np.float32))
    u = g.random(32)
    u[:4] = 0.0, 0.5, 0.25, 1 - 2.0 ** -24
    compare(cuda, x, u, k=g.integers(0, vocab + 2, 32))
    compare(cuda, x, u, p=np.tile([0.5, 0.25, 0.75, 1.0], 8), k=np.full(32, vocab // 2 * 2))
    compare(cuda, x, u, m=np.tile([0.0, 1.0, 0.4, 0.1], 8))


def test_steep_flat_and_far(cuda):
    """Temperatures from next to nothing to infinity, logits of any size."""
    g = np.random.default_rng(1)
    x = torch.from_numpy((3 * g.standard_normal((30, 3000))).astype(np.float32))
    x[10:15] *= 1e30
    x[15:20] *= 1e-30
    x[20:] -= 5e4
    t = np.tile([1e-38, 1e-20, 1e-3, 100.0, 1e30, math.inf, 1.0, 0.0, -1.0, math.nan], 3)
    compare(cuda, x, g.random(30), t=t)
    compare(cuda, x, g.random(30), t=t, k=np.full(30, 50), p=np.full(30, 0.9), m=np.full(30, 0.01))


def test_values_that_are_no_tokens(cuda):
    x = torch.full((8, 500), -math.inf)
    x[1, 77] = -3e38
    x[2] = math.nan
    x[3], x[3, 5], x[3, 7] = 0.0, math.nan, -math.inf
    x[4, 100], x[4, 400] = math.inf, math.inf
    x[5, 9], x[5, 11] = math.inf, math.nan
    x[6, 3], x[6, 2] = -0.0, 0.0
    x[7, 499] = 1e-45
    for u in (0.0, 0.3, 0.999):
        compare(cuda, x, np.full(8, u))
        compare(cuda, x, np.full(8, u), t=np.zeros(8))
        compare(cuda, x, np.full(8, u), k=np.full(8, 1), p=np.full(8, 0.1))


def test_numbers_out_of_range(cuda):
    g = np.random.default_rng(2)
    x = torch.from_numpy(g.standard_normal((7, 900)).astype(np.float32))
    u = np.array([-1.0, 1.0, 2.0, math.nan, math.inf, -math.inf, 0.5])
    compare(cuda, x, u)
    compare(cuda, x, u, p=np.array([-1, 0, 1, 2, math.nan, math.inf, 1e-30]),
            m=np.array([-1, 0, 1, 2, math.nan, math.inf, 1e-30]),
            k=np.array([-5, 0, 1, 900, 901, 2 ** 31 - 1, -2 ** 31]))


def test_draws_near_borders(cuda):
    """u * sum one step on either side of a cumulative weight."""
    n = 64
    x = torch.zeros(1, n).repeat(3 * n, 1)
    edge = np.arange(n) / n
    u = np.concatenate([edge, np.nextafter(edge, 1), np.maximum(np.nextafter(edge, 0), 0)])
    compare(cuda, x, u, wide=True)
    got, _ = run(cuda, x, u, wide=True)
    assert got[:n].tolist() == list(range(n))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("offset,stride", [(0, 1003), (1, 1008), (3, 1001), (0, 1008)])
def test_strided_rows(cuda, dtype, offset, stride):
    """Rows of a wider buffer at any alignment; what stands beside them is not
    read."""
    g = np.random.default_rng(3)
    big = torch.full((20, stride), math.inf, dtype=dtype, device=cuda)
    x = torch.from_numpy((3 * g.standard_normal((20, 997))).astype(np.float32)).to(dtype)
    big[:, offset:offset + 997] = x.to(cuda)
    view = big[:, offset:offset + 997]
    u = g.random(20)
    got = kernels.sample(view, on(u, F32, cuda), top_k=on(np.full(20, 40), I32, cuda))
    want = [plain(r, float(np.float32(v)), k=40)[0] for r, v in zip(x.float().numpy(), u)]
    assert got.tolist() == want


def test_rows_of_requests(cuda):
    """Rules by request, trees' rows; rows of no request are left."""
    g = np.random.default_rng(4)
    offsets = [2, 3, 3, 20, 21, 25]
    x = torch.from_numpy((3 * g.standard_normal((30, 2000))).astype(np.float32))
    request = [None] * 30
    for r in range(5):
        for i in range(offsets[r], offsets[r + 1]):
            request[i] = r
    q = rules(g, 5)
    u = g.random(30)
    compare(cuda, x, u, request=request, offsets=offsets, **q)
    out = torch.full((30,), -77, dtype=I32, device=cuda)
    kernels.sample(x.to(cuda), on(u, F32, cuda), offsets=on(offsets, I32, cuda), out=out)
    left = [i for i, r in enumerate(request) if r is None]
    assert out[left].tolist() == [-77] * len(left) and -77 not in out[2:25].tolist()


def test_empty(cuda):
    z = torch.zeros
    assert kernels.sample(z(0, 5, device=cuda), z(0, device=cuda)).shape == (0,)
    assert kernels.sample(z(3, 0, device=cuda), z(3, device=cuda)).tolist() == [-1] * 3
    assert kernels.sample(z(3, 5, device=cuda), z(3, device=cuda),
                          offsets=z(1, dtype=I32, device=cuda)).shape == (3,)


def test_frequencies(cuda):
    """Draws of many uniform numbers have the kept tokens' shares: each count
    within 6 standard deviations."""
    n = 20000
    x = torch.tensor([0.0, 1.0, 2.0, -1.0, 2.0]).repeat(n, 1)
    u = (np.arange(n) + 0.5) / n
    got, _ = run(cuda, x, u, t=np.full(n, 1.0), k=np.full(n, 4))
    count = np.bincount(got.cpu().numpy(), minlength=5) / n
    w = np.exp([0.0, 1.0, 2.0, -1.0, 2.0])
    w[3] = 0
    assert np.abs(count - w / w.sum()).max() <= 1.5 / n  # evenly spaced: one each side


def test_captured(cuda):
    """A graph of the draw follows its inputs, with eager work between."""
    g = np.random.default_rng(5)
    x = torch.zeros(12, 30000, device=cuda)
    u = torch.zeros(12, device=cuda)
    q = {n: torch.zeros(12, dtype=I32 if n == "top_k" else F32, device=cuda)
         for n in ("temperature", "top_k", "top_p", "min_p")}
    kernels.sample(x, u, **q)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, share = kernels.sample(x, u, probabilities=True, **q)
    for _ in range(4):
        r = rules(g, 12)
        x.copy_(torch.from_numpy((4 * g.standard_normal((12, 30000))).astype(np.float32)))
        u.copy_(torch.from_numpy(g.random(12).astype(np.float32)))
        for n, v in zip(q, (r["t"], r["k"], r["p"], r["m"])):
            q[n].copy_(torch.from_numpy(v))
        graph.replay()
        a, b = kernels.sample(x, u, probabilities=True, **q)
        torch.cuda.synchronize()
        assert torch.equal(a, got) and torch.equal(b, share)
        want = [plain(x[i].cpu().numpy(), float(u[i]), r["t"][i], r["k"][i], r["p"][i],
                      r["m"][i])[0] for i in range(12)]
        assert got.tolist() == want


def test_two_streams(cuda):
    """Calls that run at once on two streams do not meet."""
    g = np.random.default_rng(6)
    x = [torch.from_numpy((3 * g.standard_normal((6, 100000))).astype(np.float32)).to(cuda)
         for _ in range(2)]
    u = [torch.from_numpy(g.random(6).astype(np.float32)).to(cuda) for _ in range(2)]
    p = torch.full((6,), 0.9, device=cuda)
    want = [kernels.sample(a, b, top_p=p) for a, b in zip(x, u)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(kernels.sample(x[i], u[i], top_p=p))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])


def test_same_row_draws_the_same_anywhere(cuda):
    """A row alone and among many: the sums are exact."""
    g = np.random.default_rng(7)
    x = torch.from_numpy((3 * g.standard_normal((1, 128256))).astype(np.float32)).to(cuda)
    u = torch.full((1,), 0.83, device=cuda)
    one, share = kernels.sample(x, u, probabilities=True)
    for n in (2, 31, 400):
        got, chance = kernels.sample(x.expand(n, -1).contiguous(), u.expand(n).contiguous(),
                                     probabilities=True)
        assert bool((got == one).all()) and bool((chance == share).all())
