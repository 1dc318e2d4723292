"""Rotation at given positions against 64-bit rotation.

float32: the angle (64 bits) is good to 2^-28, sine and cosine to 2 units
(2^-23) of 1, products and sum add three roundings of 2^-24 of |x| + |y|:
2^-21 (|x| + |y|) scale covers them. bfloat16 adds half a step, 2^-8, of the
result."""
import math

import numpy as np
import pytest
import torch

from ncmorph_amd import decoder, kernels

pytestmark = pytest.mark.gpu


def rotate64(x, pos, inv, heads, hd, layout, scale):
    rows, half = x.shape[0], inv.numel()
    v = x[:, :heads * hd].double().reshape(rows, heads, hd).clone()
    a = pos.double()[:, None] * inv.double()[None]
    c, s = (scale * a.cos())[:, None], (scale * a.sin())[:, None]
    i = torch.arange(half)
    p, q = (i, i + half) if layout == "half" else (2 * i, 2 * i + 1)
    e, d = v[..., p].clone(), v[..., q].clone()
    v[..., p], v[..., q] = e * c - d * s, d * c + e * s
    size = torch.zeros_like(v)
    size[..., p] = size[..., q] = (e.abs() + d.abs()) * scale
    return v.reshape(rows, -1), size.reshape(rows, -1)


def check(y, x, pos, inv, heads, hd, layout, scale):
    ref, size = rotate64(x.cpu(), pos.cpu(), inv.cpu(), heads, hd, layout, scale)
    y = y.cpu()
    tol = 2.0 ** -21 * size
    if y.dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * ref.abs()
    assert bool(((y.double() - ref).abs() <= tol + 1e-38).all())
    rot = 2 * inv.numel()
    rest = y.reshape(y.shape[0], heads, hd)[..., rot:]
    assert torch.equal(rest, x.cpu()[:, :heads * hd].reshape(y.shape[0], heads, hd)[..., rot:])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,heads,hd,rot", [
    (1, 1, 64, 64), (1, 5, 128, 32), (3, 40, 128, 128), (77, 12, 64, 16), (9, 3, 80, 80),
    (5, 2, 6, 2), (7, 3, 20, 10), (4100, 4, 64, 64), (2, 1, 256, 192)])
def test_rotation(ncm, cuda, rows, heads, hd, rot, dtype, layout):
    g = torch.Generator().manual_seed(rows + rot)
    x = torch.randn(rows, heads * hd, generator=g).to(dtype).to(cuda)
    pos = torch.randint(-5, 1 << 20, (rows,), generator=g, dtype=torch.int32).to(cuda)
    inv, _ = decoder.rope_frequencies(rot, 10000.0)
    inv = torch.from_numpy(inv).to(cuda)
    y = kernels.rope_positions(x, pos, inv, heads, hd, layout=layout, scale=1.25)
    check(y, x, pos, inv, heads, hd, layout, 1.25)
    # In place, the same bits.
    z = x.clone()
    assert kernels.rope_positions(z, pos, inv, heads, hd, layout=layout, scale=1.25, out=z) is z
    assert torch.equal(z.view(torch.int16), y.view(torch.int16))


def test_far_positions_and_every_quadrant(ncm, cuda):
    """Positions to the ends of int32, and angles all around the circle."""
    ends = [0, 1, -1, 2**31 - 1, -2**31, 2**30 + 1, 131071, 1048575]
    pos = torch.tensor(ends + list(range(1, 1500)), dtype=torch.int32, device=cuda)
    g = torch.Generator().manual_seed(3)
    x = torch.randn(pos.numel(), 64, generator=g).to(cuda)
    inv = torch.from_numpy(decoder.rope_frequencies(64, 500000.0)[0]).to(cuda)
    check(kernels.rope_positions(x, pos, inv, 1, 64), x, pos, inv, 1, 64, "half", 1.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shift,wide", [(0, 200), (8, 200), (1, 201), (3, 135)])
def test_strides_and_alignment(ncm, cuda, dtype, shift, wide):
    """Column slices of a wider buffer, aligned or not; its other columns stay."""
    g = torch.Generator().manual_seed(shift)
    buf = torch.randn(6, wide, generator=g).to(dtype).to(cuda)
    x = buf[:, shift:shift + 128]
    pos = torch.arange(6, dtype=torch.int32, device=cuda) * 17
    inv = torch.from_numpy(decoder.rope_frequencies(64, 10000.0)[0]).to(cuda)
    y = kernels.rope_positions(x, pos, inv, 2, 64)
    check(y, x, pos, inv, 2, 64, "half", 1.0)
    before = buf.clone()
    kernels.rope_positions(x, pos, inv, 2, 64, out=x)
    assert torch.equal(x, y)
    assert torch.equal(buf[:, :shift], before[:, :shift])
    assert torch.equal(buf[:, shift + 128:], before[:, shift + 128:])


def test_nothing_to_do(ncm, cuda):
    inv = torch.ones(32, device=cuda)
    for rows, heads in ((0, 4), (4, 0)):
        x = torch.zeros(rows, 4 * 64, device=cuda)
        y = kernels.rope_positions(x, torch.zeros(rows, dtype=torch.int32, device=cuda), inv,
                                   heads, 64)
        assert y.shape == (rows, heads * 64)


def test_against_the_table_rotation(ncm, cuda):
    """rope_rotate at positions 0 .. n - 1: the same rotation but for its bf16
    rounding of tables, products and sum: four half steps of |x| + |y|."""
    spec = decoder.DecoderSpec(hidden=64, intermediate=64, vocab=64, q_heads=2, kv_heads=1,
                               head_dim=64, layers=1)
    cos, sin = (torch.from_numpy(t).to(cuda) for t in decoder.rope_tables(spec, 50))
    x = torch.randn(50, 128, generator=torch.Generator().manual_seed(1)).bfloat16().to(cuda)
    inv = torch.from_numpy(decoder.rope_inverse_frequencies(spec)).to(cuda)
    pos = torch.arange(50, dtype=torch.int32, device=cuda)
    y = kernels.rope_positions(x, pos, inv, 2, 64)
    z = kernels.rope_rotate(x.clone(), 2, 64, 50, cos, sin)
    _, size = rotate64(x.cpu(), pos.cpu(), inv.cpu(), 2, 64, "half", 1.0)
    assert bool(((y.double() - z.double()).abs().cpu() <= 4 * 2.0 ** -8 * size + 1e-30).all())


def test_capture(ncm, cuda):
    """A captured rotation follows the positions at replay."""
    x = torch.randn(9, 256, device=cuda)
    pos = torch.zeros(9, dtype=torch.int32, device=cuda)
    inv = torch.from_numpy(decoder.rope_frequencies(64, 10000.0)[0]).to(cuda)
    y = torch.empty_like(x)
    kernels.rope_positions(x, pos, inv, 4, 64, out=y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kernels.rope_positions(x, pos, inv, 4, 64, out=y)
    for k in range(3):
        pos.copy_(torch.arange(9, device=cuda) * (k + 1) * 1000)
        graph.replay()
        got = y.clone()
        torch.cuda.synchronize()
        assert torch.equal(got, kernels.rope_positions(x, pos, inv, 4, 64))
