"""Products with 4-bit weights (kernels.linear_int4, pack_int4, quantise_int4)
against 64-bit arithmetic.

Bound of the rounded cases: an output is s (sum (128 + q) x - (128 + z) sum x)
over groups in fp32. With E = sum_g |s| sum_k (256 + q + z) |x|, a group's sums
of at most 128 products and its difference take 130 roundings, the groups' sum
and the wavefronts' one each: (130 + groups + 8) 2^-24 E, bias and residual one
more of the result, and half a step of the output's type. Integer cases (small
integers, scales powers of two) have exact sums and are equal."""
import pytest
import torch

from ncmorph_amd import kernels

pytestmark = pytest.mark.gpu

BF16, F32, U8 = torch.bfloat16, torch.float32, torch.uint8


def up(a, b):
    return -(-a // b)


def weights(seed, n, k, group, zeros, integers=False):
    g = torch.Generator().manual_seed(seed)
    groups = up(k, group)
    codes = torch.randint(0, 16, (n, k), generator=g, dtype=U8)
    if integers:
        scales = 2.0 ** torch.randint(-1, 3, (n, groups), generator=g)
    else:
        scales = (0.5 + torch.rand(n, groups, generator=g)) * 0.02
    z = torch.randint(0, 16, (n, groups), generator=g, dtype=U8) if zeros else None
    return codes, scales.to(BF16), z


def spread(t, group, k):
    return t.double().repeat_interleave(group, 1)[:, :k]


def exact(x, codes, scales, zeros, group, bias=None, residual=None):
    """(y, E) in 64 bits."""
    k = codes.shape[1]
    z = 8.0 if zeros is None else spread(zeros, group, k)
    s = spread(scales, group, k)
    y = x[:, :k].double() @ ((codes.double() - z) * s).t()
    e = x[:, :k].double().abs() @ ((256 + codes.double() + z) * s.abs()).t()
    if bias is not None:
        y = y + bias.double()
    if residual is not None:
        y = y + residual.double()
    return y, e


def check(got, y, e, k, group, out_mode):
    half = 2.0 ** -24 if out_mode == "f32" else 2.0 ** -8
    bound = (138 + up(k, group)) * 2.0 ** -24 * e + (half + 2.0 ** -23) * y.abs() + 1e-37
    worst = ((got.double().cpu() - y).abs() / bound).max()
    assert float(worst) <= 1.0, float(worst)


SHAPES = [(1, 1, 8), (1, 16, 128), (3, 17, 136), (16, 40, 1000), (17, 33, 4096), (1, 576, 1536),
          (2, 2048, 2048), (31, 64, 14336), (33, 100, 576), (64, 257, 896), (65, 48, 264),
          (130, 1000, 512), (300, 16, 8)]


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_integers(cuda, m, n, k, group, zeros):
    """Exact sums: every code is at its place, with its scale and zero."""
    codes, scales, z = weights(m + n + k, n, k, group, zeros, integers=True)
    g = torch.Generator().manual_seed(k)
    x = torch.randint(-3, 4, (m, k), generator=g).to(BF16)
    w = kernels.pack_int4(codes.to(cuda), scales.to(cuda), group,
                          zeros=None if z is None else z.to(cuda))
    y, _ = exact(x, codes, scales, z, group)
    # Sums within a group: integers of at most 128 * 143 * 3; of groups:
    # multiples of 1 / 2 of at most 15 * 3 * 4 each.
    assert 128 * 143 * 3 < 2 ** 24 and 2 * 15 * 3 * 4 * k < 2 ** 24
    got = kernels.linear_int4(x.to(cuda), w)
    assert got.dtype == F32 and torch.equal(got.double().cpu(), y)


@pytest.mark.parametrize("out_mode", ["f32", "bf16", "bf16_f32"])
@pytest.mark.parametrize("m,n,k,group,zeros", [(1, 100, 4096, 128, False), (5, 4096, 896, 32, True),
                                               (61, 320, 14336, 64, True), (20, 51, 2056, 128, True),
                                               (200, 640, 576, 32, False)])
def test_rounded(cuda, out_mode, m, n, k, group, zeros):
    codes, scales, z = weights(1, n, k, group, zeros)
    g = torch.Generator().manual_seed(2)
    x = (torch.randn(m, k, generator=g) + 0.5).to(BF16)
    bias, residual = torch.randn(n, generator=g).to(BF16), torch.randn(m, n, generator=g)
    w = kernels.pack_int4(codes.to(cuda), scales.to(cuda), group,
                          zeros=None if z is None else z.to(cuda))
    for b, r in ((None, None), (bias, None), (None, residual), (bias, residual)):
        y, e = exact(x, codes, scales, z, group, b, r)
        got = kernels.linear_int4(x.to(cuda), w, bias=None if b is None else b.to(cuda),
                                  residual=None if r is None else r.to(cuda), out_mode=out_mode)
        assert got.dtype == (BF16 if out_mode == "bf16" else F32)
        check(got, y, e, k, group, out_mode)
    if out_mode != "bf16":
        into = residual.to(cuda)
        assert kernels.linear_int4(x.to(cuda), w, residual=into, out=into, out_mode=out_mode) is into
        y, e = exact(x, codes, scales, z, group, None, residual)
        check(into, y, e, k, group, out_mode)


@pytest.mark.parametrize("m,n,k,group,zeros", [
    (4, 52437, 136, 32, True), (5, 52437, 136, 64, False), (9, 29131, 264, 128, True),
    (16, 16384, 520, 32, True), (16, 16385, 520, 32, True), (16, 16401, 2056, 128, False)])
def test_few_rows_of_many_outputs(cuda, m, n, k, group, zeros):
    """Either side of 2^18 outputs in all, where rows begin to be shared."""
    codes, scales, z = weights(n + k, n, k, group, zeros)
    g = torch.Generator().manual_seed(m)
    x, bias = torch.randn(m, k, generator=g).to(BF16), torch.randn(n, generator=g).to(BF16)
    residual = torch.randn(m, n, generator=g)
    w = kernels.pack_int4(codes.to(cuda), scales.to(cuda), group,
                          zeros=None if z is None else z.to(cuda))
    y, e = exact(x, codes, scales, z, group, bias, residual)
    out = residual.to(cuda)
    got = kernels.linear_int4(x.to(cuda), w, bias=bias.to(cuda), residual=out, out=out)
    assert got.data_ptr() == out.data_ptr()
    # Bias and residual round at the size of the terms, not of the sum.
    check(got, y, e + 0.5 * (bias.abs() + residual.abs()).double(), k, group, "f32")


@pytest.mark.parametrize("n", [31, 32])
@pytest.mark.parametrize("out_mode", ["f32", "bf16"])
def test_strides_and_alignment(cuda, n, out_mode):
    """Columns of a wider x, outputs and bias at odd addresses; nothing beside
    the output changes."""
    m, k, group = 19, 520, 64
    codes, scales, _ = weights(3, n, k, group, False, integers=True)
    wide = torch.full((m, 1600), float("nan")).to(BF16)
    x = torch.randint(-3, 4, (m, k)).to(BF16)
    wide[:, 8:8 + k] = x
    wide = wide.to(cuda)
    w = kernels.pack_int4(codes.to(cuda), scales.to(cuda), group)
    dt = F32 if out_mode == "f32" else BF16
    store = torch.full((m * n + 9,), -5.0, dtype=dt, device=cuda)
    bias = torch.randint(-3, 4, (n + 1,)).to(BF16).to(cuda)[1:]
    out = store[1:1 + m * n].view(m, n)
    kernels.linear_int4(wide[:, 8:8 + k], w, bias=bias, out=out, out_mode=out_mode)
    y, _ = exact(x, codes, scales, None, group, bias.cpu())
    assert torch.equal(out.cpu(), y.float().to(dt))
    assert float(store[0]) == -5.0 and bool((store[1 + m * n:] == -5.0).all())


def test_a_bad_row_stays_alone(cuda):
    """NaN and infinities in one row of x, a NaN scale of one output."""
    m, n, k = 35, 48, 256
    codes, scales, _ = weights(4, n, k, 32, False, integers=True)
    x = torch.randint(-3, 4, (m, k)).to(BF16)
    y, _ = exact(x, codes, scales, None, 32)
    bad = x.clone()
    bad[3, 200], bad[17, 0], bad[34, 255] = float("nan"), float("inf"), -float("inf")
    scales[7, 2] = float("nan")
    w = kernels.pack_int4(codes.to(cuda), scales.to(cuda), 32)
    got = kernels.linear_int4(bad.to(cuda), w).double().cpu()
    rows = [i for i in range(m) if i not in (3, 17, 34)]
    cols = [j for j in range(n) if j != 7]
    assert torch.equal(got[rows][:, cols], y[rows][:, cols])
    assert bool(got[[3, 17, 34]].isnan().all()) and bool(got[:, 7].isnan().all())


def test_empty(cuda):
    codes, scales, _ = weights(5, 20, 64, 32, False)
    w = kernels.pack_int4(codes.to(cuda), scales.to(cuda), 32)
    assert kernels.linear_int4(torch.zeros(0, 64, dtype=BF16, device=cuda), w).shape == (0, 20)
    none = kernels.pack_int4(torch.zeros(0, 64, dtype=U8, device=cuda),
                             torch.zeros(0, 2, dtype=BF16, device=cuda), 32)
    assert kernels.linear_int4(torch.zeros(3, 64, dtype=BF16, device=cuda), none).shape == (3, 0)


def plain_quantise(w, group, symmetric):
    """Float32, as documented."""
    n, k = w.shape
    groups = up(k, group)
    x = torch.zeros(n, groups * group)
    x[:, :k] = w.float()
    x = x.view(n, groups, group)
    bad = ~torch.isfinite(x).all(-1)
    safe = torch.where(bad[..., None], torch.zeros(()), x)
    lo, hi = safe.amin(-1).clamp(max=0), safe.amax(-1).clamp(min=0)
    unit = torch.maximum(hi, -lo) / 7 if symmetric else hi / 15 - lo / 15
    scale = torch.where(bad, torch.tensor(float("nan")), unit).to(BF16)
    s = scale.float()
    none = bad | (s == 0)
    div = torch.where(none, torch.ones(()), s)
    z = torch.full((n, groups), 8.0)
    if not symmetric:
        z = torch.where(none, z, torch.round(-lo / div).clamp(0, 15))
    q = (torch.round(safe / div[..., None]) + z[..., None]).clamp(0, 15)
    q = torch.where(none[..., None], z[..., None], q)
    return q.view(n, -1)[:, :k].to(U8), scale, z.to(U8)


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,k", [(1, 8), (5, 136), (100, 1000), (33, 4096)])
def test_quantise(cuda, n, k, group, symmetric):
    g = torch.Generator().manual_seed(n + k)
    w = (torch.randn(n, k, generator=g) * 10 ** (3 * torch.rand(n, 1, generator=g))).to(BF16)
    w[0, :8] = 0
    if n > 3:
        w[1], w[2, k // 2], w[3, 0] = 0, float("nan"), float("inf")
        w[4] = w[4].abs()
        w[n - 1, :3] = torch.tensor([3.3e38, -3.3e38, 1e-40]).to(BF16)
    wide = torch.zeros(n, k + 5, dtype=BF16)
    wide[:, 5:] = w
    codes, scales, zeros = kernels.quantise_int4(wide.to(cuda)[:, 5:], group, symmetric)
    q, s, z = plain_quantise(w, group, symmetric)
    assert torch.equal(codes.cpu(), q)
    assert torch.equal(scales.cpu().isnan(), s.isnan())
    assert torch.equal(scales.cpu().nan_to_num(-1.0), s.nan_to_num(-1.0))
    assert zeros is None if symmetric else torch.equal(zeros.cpu(), z)


def test_quantised_products(cuda):
    """From bf16 weights to products: within the codes' half steps of x |w|'s
    exact product (a clamped code, which the scale's rounding allows for the
    largest weights, is 7 * 2^-8 of a step further)."""
    n, k, group, m = 300, 2048, 128, 7
    g = torch.Generator().manual_seed(6)
    w, x = torch.randn(n, k, generator=g).to(BF16), torch.randn(m, k, generator=g).to(BF16)
    codes, scales, _ = kernels.quantise_int4(w.to(cuda), group)
    packed = kernels.pack_int4(codes, scales, group)
    got = kernels.linear_int4(x.to(cuda), packed).double().cpu()
    _, e = exact(x, codes.cpu(), scales.cpu(), None, group)
    step = x.double().abs() @ spread(scales.cpu(), group, k).t()
    assert bool(((got - x.double() @ w.double().t()).abs()
                 <= (0.5 + 7 * 2.0 ** -8) * step + 200 * 2.0 ** -24 * e).all())


def test_captured_and_other_streams(cuda):
    """Bit for bit the same in a graph, with eager work between replays, and on
    another stream."""
    codes, scales, z = weights(7, 500, 1024, 64, True)
    w = kernels.pack_int4(codes.to(cuda), scales.to(cuda), 64, zeros=z.to(cuda))
    x = torch.zeros(9, 1024, dtype=BF16, device=cuda)
    kernels.linear_int4(x, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = kernels.linear_int4(x, w)
    side = torch.cuda.Stream()
    for i in range(4):
        x.copy_(torch.randn(9, 1024, generator=torch.Generator().manual_seed(i)))
        graph.replay()
        ref = kernels.linear_int4(x, w)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = kernels.linear_int4(x, w)
        torch.cuda.synchronize()
        assert torch.equal(got, ref) and torch.equal(other, ref)
