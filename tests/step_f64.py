"""Plain 64-bit forms of the operators that continue a sequence, on the CPU,
and small steps to run them on: requests of given new rows and tokens before
them over a paged cache whose unused places hold NaN."""
import math

import numpy as np
import torch

BF16, FP8, I8 = torch.bfloat16, torch.float8_e4m3fn, torch.int8


def quantise(x, dtype):
    """(codes, scales) of the last dimension's rows, from exact arithmetic."""
    if dtype == BF16:
        return x.clone(), None
    x = x.double()
    m = x.abs().amax(-1, keepdim=True)
    bad = ~torch.isfinite(x).all(-1, keepdim=True)
    x, m = torch.where(bad, 0.0, x), torch.where(bad, 0.0, m)
    if dtype == I8:
        codes = torch.round(x * 127.0 / torch.where(m > 0, m, 1.0)).to(I8)
        scale = (m.float() / 127.0).double()
    else:
        f, e = np.frexp((m / 448.0).numpy())
        e = np.maximum(e - (f == 0.5), -126)                 # ceil(log2), exactly
        scale = torch.from_numpy(np.ldexp(1.0, np.where(m.numpy() > 0, e, -126)))
        codes = (x / scale).float().to(FP8)                  # exact in float32, one rounding
    scale = torch.where(bad, math.nan, scale)
    return codes, scale[..., 0].float()


def values(codes, scales):
    v = codes.to(torch.float32).double()
    return v if scales is None else v * scales.double()[..., None]


class Step:
    """Requests with `new` rows after `before` tokens; K and V of all their
    tokens lie in the cache's pages, in any order, everything else there is NaN
    (bf16), the NaN code (fp8) or a NaN scale."""

    def __init__(self, seed, new, before, kv_heads, hd, page, dtype, extra_rows=0, spare=2,
                 cache_of=None):
        g = torch.Generator().manual_seed(seed)
        self.new, self.before, self.page, self.dtype = list(new), list(before), page, dtype
        self.heads, self.hd = kv_heads, hd
        self.rows = sum(new) + extra_rows
        self.offsets = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32)
        self.starts = torch.tensor(before, dtype=torch.int32)
        need = [-(-(n + c) // page) for n, c in zip(new, before)]
        total = sum(need) + spare
        order = torch.randperm(total, generator=g).int()
        self.table = torch.full((len(new), max(need + [0]) + 1), -1, dtype=torch.int32)
        at = 0
        for r, n in enumerate(need):
            self.table[r, :n] = order[at:at + n]
            at += n
        shape = (total, kv_heads, page, hd)
        self.tokens, self.pages, self.scales = [], [], []
        for _ in range(2):
            dense = [torch.randn(n + c, kv_heads, hd, generator=g).to(BF16)
                     for n, c in zip(new, before)]
            if dtype == BF16:
                pages, scales = torch.full(shape, math.nan, dtype=BF16), None
            else:
                fill = torch.full(shape, 127, dtype=torch.uint8).view(dtype)  # e4m3: NaN
                pages, scales = fill, torch.full(shape[:3], math.nan)
            for r, x in enumerate(dense):
                codes, sc = quantise(x, dtype)
                for t in range(x.shape[0]):
                    p = int(self.table[r, t // page])
                    pages.view(torch.uint8 if dtype != BF16 else BF16)[p, :, t % page] = (
                        codes[t].view(torch.uint8) if dtype != BF16 else codes[t])
                    if sc is not None:
                        scales[p, :, t % page] = sc[t]
            self.tokens.append(dense)
            self.pages.append(pages)
            self.scales.append(scales)

    def to(self, device):
        """(KvCache, page_table, offsets, starts) on the device."""
        from ncmorph_amd import cache

        on = [None if t is None else t.to(device) for t in self.pages + self.scales]
        kv = cache.KvCache(*on)
        return kv, self.table.to(device), self.offsets.to(device), self.starts.to(device)

    def cached(self, which):
        """What the cache stands for of every request's tokens, in 64 bits."""
        return [values(*quantise(x, self.dtype)) for x in self.tokens[which]]


def chain(new):
    """[n, n] allowed pairs of each request's rows: its own and earlier ones."""
    return [torch.ones(n, n).tril().bool() for n in new]


def tree(seed, new):
    """Ancestors and itself, of random trees."""
    rng = np.random.default_rng(seed)
    out = []
    for n in new:
        a = torch.eye(n).bool()
        for i in range(1, n):
            a[i] |= a[int(rng.integers(0, i))]
        out.append(a)
    return out


def bits(allowed, rows, words):
    """int64 [rows, words] of per-request pairs; rows of no request all ones."""
    m = np.full((rows, words), -1, np.int64).view(np.uint64)
    at = 0
    for a in allowed:
        for i in range(a.shape[0]):
            m[at + i] = 0
            for j in np.flatnonzero(a[i].numpy()):
                if j < 64 * words:
                    m[at + i, j // 64] |= np.uint64(1) << np.uint64(j % 64)
        at += a.shape[0]
    return torch.from_numpy(m.view(np.int64))


def attention(step, q, q_heads, allowed, window=0, positions=None, scale=None, missing=(),
              chained=False):
    """(outputs, sum of p |v|) [rows, q_heads, hd] in 64 bits; rows of no
    request NaN. chained: no mask, so the window holds for new rows too.
    `missing`: (request, page index) whose tokens are not there."""
    group, hd = q_heads // step.heads, step.hd
    scale = hd ** -0.5 if scale is None else scale
    out = torch.full((step.rows, q_heads, hd), math.nan, dtype=torch.float64)
    mag = out.clone()
    K, V = step.cached(0), step.cached(1)
    at = 0
    for r, (n, c) in enumerate(zip(step.new, step.before)):
        for i in range(n):
            see = torch.zeros(n + c, dtype=torch.bool)
            see[:c] = True
            if window:
                p = c + i if positions is None else max(int(positions[at + i]), c)
                see[:c] = torch.arange(c) > p - window
            if window and chained:
                see = (torch.arange(n + c) > p - window) & (torch.arange(n + c) <= c + i)
            else:
                see[c:] = allowed[r][i]
            for rr, page in missing:
                if rr == r:
                    see[page * step.page:(page + 1) * step.page] = False
            keys = torch.nonzero(see)[:, 0]
            for h in range(q_heads):
                k, v = K[r][keys, h // group], V[r][keys, h // group]
                if not len(keys):
                    out[at + i, h], mag[at + i, h] = 0.0, 0.0
                    continue
                s = (k @ q[at + i, h * hd:(h + 1) * hd].double()) * scale
                w = torch.softmax(s, 0)
                out[at + i, h], mag[at + i, h] = w @ v, w @ v.abs()
        at += n
    return out, mag


def attention_bound(ref, mag):
    """The output's own rounding (2^-8), and 2^-10 of sum p |v| for the fp32
    scores (130 roundings of 2^-24 of sum |q k|), exponentials, sums and
    probabilities of two bf16 terms (2^-16)."""
    return 2.0 ** -10 * mag + 2.0 ** -8 * ref.abs() + 1e-30
