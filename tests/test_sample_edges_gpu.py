"""Token sampling (kernels.sample) where its searches end: infinite and largest
temperatures, distances that fp32 does not hold, cuts among the least weights,
draws one step from a border; by test_sample_gpu's plain form."""
import math

import numpy as np
import pytest
import torch

from tests.test_sample_gpu import BF16, F32, compare

pytestmark = pytest.mark.gpu

BIG = 3.3e38


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [6, 1000, 40000])
def test_infinite_temperatures_and_distances(cuda, dtype, vocab):
    """Every token there weighs the same at a temperature of infinity: rows of
    forced tokens, and values further from the largest than fp32 goes."""
    x = torch.full((8, vocab), -math.inf)
    x[0, 4] = math.inf
    x[1, 2], x[1, vocab - 1] = math.inf, math.inf
    x[2, 1], x[2, 3], x[2, 5] = BIG, -BIG, 0.0
    x[3, 0], x[3, 5] = math.inf, -BIG
    x[4, 3], x[4, 4] = -BIG, math.nan
    x[5] = -BIG
    x[5, 2] = BIG
    x[6], x[6, 1] = 0.0, math.inf
    x[7, 2], x[7, 4] = 1e30, -1e30
    x = x.to(dtype)
    inf = np.full(8, math.inf)
    for u in (0.0, 0.3, 0.6, 1 - 2.0 ** -24):
        u = np.full(8, u)
        compare(cuda, x, u, t=inf)
        compare(cuda, x, u, t=inf, k=np.full(8, 2))
        compare(cuda, x, u, t=inf, p=np.full(8, 0.7), m=np.full(8, 1.0))
        compare(cuda, x, u, t=inf, k=np.full(8, 5), p=np.full(8, 0.9), m=np.full(8, 0.3))


@pytest.mark.parametrize("least", [0.05, 0.13, 0.14, 0.5])
def test_largest_temperatures(cuda, least):
    """exp(-2 * 3.3 / 3.4) = 0.143 is the weight of the farthest token there
    can be: min_p and top_p on either side of it."""
    x = torch.zeros(4, 500)
    x[0], x[0, 7] = -BIG, BIG
    x[1, :250], x[1, 9] = -BIG, BIG
    x[2, 250:], x[2, 9] = BIG, -BIG
    x[3, 3], x[3, 4] = math.inf, -BIG
    t = np.full(4, np.finfo(np.float32).max)
    for u in (0.0, 0.4, 0.9, 1 - 2.0 ** -24):
        u = np.full(4, u)
        compare(cuda, x, u, t=t)
        compare(cuda, x, u, t=t, m=np.full(4, least))
        compare(cuda, x, u, t=t, p=np.full(4, 0.8), m=np.full(4, least))


def test_cuts_among_the_least_weights(cuda):
    """min_p next to 2^-43, the unit of the weights: the tokens whose rounded
    weights reach it, 900 to a row, drawn from the row's very end."""
    g = np.random.default_rng(1)
    x = -np.concatenate([np.full((3, 900), 30.2), g.uniform(27, 30.4, (45, 900))]).astype(np.float32)
    x[:, 450] = 0
    m = np.concatenate([[1e-13, 1.1368e-13, 1.14e-13], 10 ** g.uniform(-14, -11.5, 45)])
    for back in (0, 40, 400):
        u = np.full(48, 1 - (1 + back) * 2.0 ** -44)
        compare(cuda, torch.from_numpy(x), u, m=m, wide=True)
        compare(cuda, torch.from_numpy(x), u, m=m, k=np.full(48, 901), wide=True)


@pytest.mark.parametrize("n", [3, 7, 11, 100, 999, 40000])
def test_draws_a_step_from_a_border(cuda, n):
    """n equal tokens and 64-bit numbers next to k / n, whose last bits are below
    2^-53 where k / n is small."""
    edge = np.unique(np.arange(n) * 64 // max(n, 64) / n) if n > 200 else np.arange(n) / n
    u = np.concatenate([edge, np.nextafter(edge, 1), np.maximum(np.nextafter(edge, 0), 0),
                        edge[1:] * (1 + 2.0 ** -50), edge[1:] * 2.0 ** -20])
    compare(cuda, torch.zeros(1, n).repeat(len(u), 1), u, wide=True)
