"""Writing the paged cache and reading it back: codes and scales bit for bit
against exact arithmetic (a bf16 value times 127 and a power of two are exact,
so one rounding is left, the same one in 32 and 64 bits), values after one
rounding to bf16."""
import math

import pytest
import torch

from ncmorph_amd import cache
from ncmorph_amd._lib import NcmError
from tests import step_f64 as f64
from tests.step_f64 import BF16, FP8, I8

pytestmark = pytest.mark.gpu

DTYPES = [BF16, FP8, I8]


def raw(t):
    return t.cpu().view(torch.int16 if t.element_size() == 2 else
                        torch.uint8 if t.element_size() == 1 else torch.int32)


def empty_like_step(step, cuda):
    """The step's cache with every byte 0xA5."""
    def fill(t):
        return (t.view(torch.uint8) * 0 + 0xA5).view(t.dtype).to(cuda) if t is not None else None
    t = [fill(x) for x in step.pages + step.scales]
    return cache.KvCache(*t), [x.clone() for x in t if x is not None]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new,before,heads,page", [
    ([1], [0], 1, 16), ([1, 1, 1], [0, 15, 16], 2, 16), ([5, 0, 40, 1], [30, 7, 0, 63], 3, 32),
    ([130], [1], 8, 1024), ([3] * 70, list(range(70)), 1, 16), ([4099, 3], [5, 0], 1, 64)])
def test_write_and_read(ncm, cuda, dtype, hd, new, before, heads, page):
    step = f64.Step(7, new, before, heads, hd, page, dtype, extra_rows=2)
    kv, table, offs, starts = step.to(cuda)
    blank, was = empty_like_step(step, cuda)
    # The step's rows as columns of one wider buffer.
    width = heads * hd
    buf = torch.full((step.rows, 3 * width), math.nan, dtype=BF16)
    for w in range(2):
        at = 0
        for x, n in zip(step.tokens[w], step.new):
            buf[at:at + n, (w + 1) * width:(w + 2) * width] = x[x.shape[0] - n:].reshape(n, width)
            at += n
    buf = buf.to(cuda)
    k, v = buf[:, width:2 * width], buf[:, 2 * width:]
    cache.write(blank, k, v, table, offs, starts)
    # Written places hold the codes, all others what they held.
    for got, want, old in zip((blank.k, blank.v, blank.k_scale, blank.v_scale),
                              step.pages + step.scales, was + [None, None]):
        if want is None:
            continue
        want, got, old = raw(want), raw(got), raw(old).clone()
        for r, (n, c) in enumerate(zip(new, before)):
            for t in range(c, c + n):
                p = int(step.table[r, t // page])
                old[p, :, t % page] = want[p, :, t % page]
        assert torch.equal(got, old)
    # Read back, into columns of a buffer: rows of no request and the other
    # columns as they were.
    out = torch.full((step.rows, 2 * width + 8), 3.0, dtype=BF16, device=cuda)
    cache.read(kv, table, offs, starts, step.rows, out=(out[:, :width], out[:, width + 8:]))
    k2, v2 = cache.read(kv, table, offs, starts, step.rows)
    want = torch.full((step.rows, 2 * width + 8), 3.0, dtype=BF16)
    for w, at0 in enumerate((0, width + 8)):
        at = 0
        for x, n in zip(step.cached(w), new):
            # float32 product, exact or rounded once, then one rounding to bf16.
            want[at:at + n, at0:at0 + width] = x[x.shape[0] - n:].reshape(n, width).float().to(BF16)
            at += n
    assert torch.equal(out.cpu(), want)
    made = sum(new)
    assert torch.equal(k2.cpu()[:made], want[:made, :width])
    assert torch.equal(v2.cpu()[:made], want[:made, width + 8:])


@pytest.mark.parametrize("dtype", [FP8, I8])
def test_rounding_edges(ncm, cuda, dtype):
    """Ties (x = m / 2), largest and smallest magnitudes, zeros, values that are
    not finite; 448 and 127 times a power of two."""
    rows = [[1.0, 0.5, -0.5, 0.25, 2.0 ** -9, 3.0], [448.0, 232.0, -1.0625, 17.0, 0.0, 1e-3],
            [450.0, 448.0, 225.0, -224.0, 1.0, 2.0], [127.0, 63.5, -62.5, 0.5, 1.5, -126.5],
            [2.0 ** 127 * 1.9921875, 2.0 ** 126, -2.0 ** 120, 1.0, 0.0, -0.0], [0.0] * 6,
            [2.0 ** -120, -2.0 ** -121, 2.0 ** -126, 0.0, 2.0 ** -123, 2.0 ** -130],
            [math.inf, 1.0, 2.0, 0.0, -1.0, 5.0], [-math.inf, 1.0, 2.0, 0.0, -1.0, 5.0],
            [1.0, math.nan, 2.0, 0.0, -1.0, 5.0]]
    x = torch.zeros(len(rows), 64)
    x[:, :6] = torch.tensor(rows)
    x = x.to(BF16)
    kv = cache.allocate(2, 1, 16, 64, dtype, cuda)
    table = torch.tensor([[1]], dtype=torch.int32, device=cuda)
    offs = torch.tensor([0, len(rows)], dtype=torch.int32, device=cuda)
    starts = torch.zeros(1, dtype=torch.int32, device=cuda)
    cache.write(kv, x.to(cuda), x.flip(1).contiguous().to(cuda), table, offs, starts)
    codes, scales = f64.quantise(x, dtype)
    n = len(rows)
    assert torch.equal(raw(kv.k)[1, 0, :n], raw(codes))
    got = kv.k_scale.cpu()[1, 0, :n]
    assert torch.equal(torch.isnan(got), torch.isnan(scales))
    fine = ~torch.isnan(scales)
    assert torch.equal(got[fine], scales[fine])
    assert torch.equal(raw(kv.v)[1, 0, :n], raw(codes.view(torch.uint8).flip(1)))
    assert int(raw(kv.k)[0].abs().sum()) == 0          # the other page
    k, _ = cache.read(kv, table, offs, starts, n)
    want = f64.values(codes, scales).float().to(BF16)
    assert torch.equal(torch.isnan(k.cpu()), torch.isnan(want))
    assert torch.equal(k.cpu()[fine], want[fine])


@pytest.mark.parametrize("dtype", DTYPES)
def test_tokens_that_are_not_there(ncm, cuda, dtype):
    """Entries of the table outside the cache, tokens past the table, offsets
    past the rows, starts below zero: left out of a write, zeros in a read."""
    step = f64.Step(11, [20, 20, 3], [0, 4, 0], 2, 64, 16, dtype)
    kv, table, offs, starts = step.to(cuda)
    pages = step.pages[0].shape[0]
    table = table[:, :2].clone()           # request 1's tokens 16 .. 23 in page 1, none past 32
    table[0, 1] = pages                    # outside
    table[1, 0] = -7
    table[2, 0] = 2**31 - 1
    starts = torch.tensor([0, 14, -3], dtype=torch.int32, device=cuda)   # request 1: 14 .. 33
    offs = torch.tensor([0, 20, 40, 1000], dtype=torch.int32, device=cuda)
    x = torch.ones(43, 128, dtype=BF16, device=cuda)
    blank = cache.allocate(pages, 2, 16, 64, dtype, cuda)
    cache.write(blank, x, x, table, offs, starts)
    k, v = cache.read(blank, table, offs, starts, 43)
    there = torch.zeros(43, dtype=torch.bool)
    there[:16] = True                      # request 0's first page
    there[22:38] = True                    # request 1's tokens 16 .. 31
    one = torch.ones(()) if dtype != I8 else (torch.tensor(127.0) * (torch.ones(()) / 127.0))
    for t in (k, v):
        assert torch.equal(t.cpu(), torch.where(there[:, None], one.to(BF16), 0.0).to(BF16)
                           .expand(43, 128))
    wrote = int((raw(blank.k) != 0).any(-1).sum())
    assert wrote == int(there.sum()) * 2


@pytest.mark.parametrize("offsets", [[3, 1, 5], [0, 6, 2], [-4, 2, 5], [5, 5, 5], [9, 9, 9]])
def test_offsets_out_of_order_stay_in_bounds(ncm, cuda, offsets):
    kv = cache.allocate(4, 1, 16, 64, BF16, cuda)
    x = torch.ones(5, 64, dtype=BF16, device=cuda)
    table = torch.tensor([[0], [1]], dtype=torch.int32, device=cuda)
    offs = torch.tensor(offsets, dtype=torch.int32, device=cuda)
    starts = torch.zeros(2, dtype=torch.int32, device=cuda)
    cache.write(kv, x, x, table, offs, starts)
    cache.read(kv, table, offs, starts, 5)
    torch.cuda.synchronize()
    assert int((raw(kv.k)[2:] != 0).sum()) == 0


def test_layers_in_one_buffer(ncm, cuda):
    """A layer's K and V as parts of [pages, layers, 2, heads, page, hd]: the
    other parts stay."""
    buf = torch.zeros(5, 3, 2, 2, 16, 64, dtype=I8, device=cuda)
    sc = torch.zeros(5, 3, 2, 2, 16, device=cuda)
    kv = cache.KvCache(buf[:, 1, 0], buf[:, 1, 1], sc[:, 1, 0], sc[:, 1, 1])
    x = torch.randn(30, 128, device=cuda, generator=torch.Generator(cuda).manual_seed(1)).to(BF16)
    table = torch.tensor([[4, 2]], dtype=torch.int32, device=cuda)
    offs = torch.tensor([0, 30], dtype=torch.int32, device=cuda)
    starts = torch.zeros(1, dtype=torch.int32, device=cuda)
    cache.write(kv, x, x.flip(0).contiguous(), table, offs, starts)
    k, v = cache.read(kv, table, offs, starts, 30)
    assert torch.equal(k, v.flip(0))
    codes, scales = f64.quantise(x.cpu().reshape(30, 2, 64), I8)
    assert torch.equal(k.cpu(), f64.values(codes, scales).float().to(BF16).reshape(30, 128))
    for layer in (0, 2):
        assert int(buf[:, layer].abs().sum()) == 0 and float(sc[:, layer].abs().sum()) == 0.0


def test_a_place_past_32_bits(ncm, cuda):
    """A page whose first code lies beyond 2^32 elements of the cache."""
    pages = (2**32 // (8 * 1024 * 128)) + 2
    kv = cache.KvCache(*(torch.empty(pages, 8, 1024, 128, dtype=I8, device=cuda) for _ in range(2)),
                       *(torch.empty(pages, 8, 1024, device=cuda) for _ in range(2)))
    x = torch.randn(3, 1024, device=cuda, generator=torch.Generator(cuda).manual_seed(1)).to(BF16)
    table = torch.tensor([[pages - 1]], dtype=torch.int32, device=cuda)
    offs = torch.tensor([0, 3], dtype=torch.int32, device=cuda)
    starts = torch.tensor([1000], dtype=torch.int32, device=cuda)
    cache.write(kv, x, x, table, offs, starts)
    codes, scales = f64.quantise(x.cpu().reshape(3, 8, 128), I8)
    assert torch.equal(kv.k[pages - 1, :, 1000:1003].cpu(), codes.permute(1, 0, 2))
    assert torch.equal(kv.v_scale[pages - 1, :, 1000:1003].cpu(), scales.t())
    k, _ = cache.read(kv, table, offs, starts, 3)
    assert torch.equal(k.cpu(), f64.values(codes, scales).float().to(BF16).reshape(3, 1024))
    # The attention over that place: one token sees itself and two before it.
    q = torch.randn(3, 1024, device=cuda, generator=torch.Generator(cuda).manual_seed(2)).to(BF16)
    mask = torch.tensor([[1], [3], [7]], dtype=torch.int64, device=cuda)
    o = cache.attention(q, kv, 8, table, offs, starts, tree_mask=mask, window=1)
    v64 = f64.values(codes, scales)
    for i in range(3):
        s = (v64[:i + 1] * q[i].cpu().double().reshape(8, 128)).sum(-1) * 128 ** -0.5
        w = torch.softmax(s, 0)[..., None]
        ref, mag = (w * v64[:i + 1]).sum(0), (w * v64[:i + 1].abs()).sum(0)
        err = (o[i].cpu().double().reshape(8, 128) - ref).abs()
        assert bool((err <= f64.attention_bound(ref, mag)).all())


def test_capture(ncm, cuda):
    """A captured write and read follow starts and the table at replay."""
    kv = cache.allocate(6, 2, 16, 64, I8, cuda)
    x = torch.zeros(4, 128, dtype=BF16, device=cuda)
    table = torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32, device=cuda)
    offs = torch.tensor([0, 2, 4], dtype=torch.int32, device=cuda)
    starts = torch.zeros(2, dtype=torch.int32, device=cuda)
    out = tuple(torch.empty(4, 128, dtype=BF16, device=cuda) for _ in range(2))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.write(kv, x, x, table, offs, starts)
        cache.read(kv, table, offs, starts, 4, out=out)
    for t in range(3):
        x.copy_(torch.randn(4, 128, device=cuda))
        starts.fill_(7 * t)
        table.copy_(table.flip(0))
        graph.replay()
        torch.cuda.synchronize()
        codes, scales = f64.quantise(x.cpu().reshape(4, 2, 64), I8)
        want = f64.values(codes, scales).float().to(BF16).reshape(4, 128)
        assert torch.equal(out[0].cpu(), want) and torch.equal(out[1].cpu(), want)


def test_nothing_to_do(ncm, cuda):
    kv = cache.allocate(1, 1, 16, 64, BF16, cuda)
    i32 = dict(dtype=torch.int32, device=cuda)
    x = torch.zeros(2, 64, dtype=BF16, device=cuda)
    none = torch.zeros(0, 1, **i32), torch.zeros(1, **i32), torch.zeros(0, **i32)
    cache.write(kv, x, x, *none)
    cache.read(kv, *none, 2)
    one = torch.zeros(1, 1, **i32), torch.zeros(2, **i32), torch.zeros(1, **i32)
    cache.write(kv, x[:0], x[:0], *one)
    assert cache.read(kv, *one, 0)[0].shape == (0, 64)
    # A table of no pages: nothing is there.
    flat = torch.zeros(1, 0, **i32), torch.tensor([0, 2], **i32), torch.zeros(1, **i32)
    cache.write(kv, x + 1, x + 1, *flat)
    assert int(kv.k.abs().sum()) == 0
    assert float(cache.read(kv, *flat, 2)[0].abs().sum()) == 0.0


def test_refused_by_the_library(ncm, cuda):
    """Alignment, which the wrapper leaves to the C ABI."""
    kv = cache.allocate(1, 1, 16, 64, BF16, cuda)
    buf = torch.zeros(2, 136, dtype=BF16, device=cuda)
    i32 = dict(dtype=torch.int32, device=cuda)
    args = torch.zeros(1, 1, **i32), torch.tensor([0, 2], **i32), torch.zeros(1, **i32)
    for bad in (buf[:, 1:65], buf[:, 4:68], torch.zeros(2, 65, dtype=BF16, device=cuda)[:, :64]):
        with pytest.raises(NcmError):
            cache.write(kv, bad, buf[:, :64], *args)
        with pytest.raises(NcmError):
            cache.read(kv, *args, 2, out=(buf[:, :64], bad))
