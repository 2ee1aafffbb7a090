"""4-bit weights in groups on the GPU: codes and back bit for bit against the
scheme's arithmetic, Linear on them against 64 bits."""
import pytest
import torch

import _w4 as W

pytestmark = pytest.mark.gpu


def _gh():
    import ghostflow_hip
    return ghostflow_hip


@pytest.mark.parametrize("n,k,group", [(1, 32, 32), (7, 96, 32), (33, 416, 64), (5, 4096, 128), (3, 1000 * 32, 256),
                                       (9, 320, 320), (4, 2080, 1024), (6, 672, 96), (2, 64, 4096)])
@pytest.mark.parametrize("symmetric", [True, False])
def test_quantize_and_back(torch_dev, n, k, group, symmetric):
    gh = _gh()
    g = torch.Generator().manual_seed(k + group)
    w = torch.randn(n, k, generator=g) * 0.02
    w[0, :32] = 0.0                       # a group without a range (group 32)
    w[-1] = w[-1].abs() + 0.01            # one sign only
    w[n // 2, ::3] *= -1
    w[:, 1] = torch.where(w[:, 1] == 0, 0.5, w[:, 1])
    want = W.quantize(w, group, symmetric)
    got = gh.quantize_grouped_i4(w.to(torch_dev), group, symmetric=symmetric)
    for a, b in zip(got, want):
        assert (a is None) == (b is None)
        if a is not None:
            assert torch.equal(a.cpu(), b)
    back = gh.dequantize_grouped_i4(*got, group).cpu()
    assert torch.equal(back, W.weight(*want, group).float())
    # no further from the weight than half a step, where no code was clamped;
    # the largest magnitude of a symmetric group is 7 steps, of an asymmetric
    # one at most a step beyond the zero point's rounding
    step = W.spread(want[1], k, group)
    assert (back - w).abs().le(step * (0.5 if symmetric else 1.0) * (1 + 2 ** -20)).all()


@pytest.mark.parametrize("symmetric", [True, False])
def test_quantize_ties_and_their_neighbours(torch_dev, symmetric):
    """Values at, next to and near half steps, for scales from 2^-140 to 2^120."""
    gh = _gh()
    g = torch.Generator().manual_seed(12)
    rows = []
    for e in (-140, -126, -101, -100, -99, -20, 0, 3, 60, 99, 100, 101, 120):
        top = (torch.rand(1, generator=g) + 1) * 7 * 2.0 ** e
        s = top * torch.tensor(1 / 7, dtype=torch.float32) if symmetric else top * torch.tensor(1 / 15, dtype=torch.float32)
        half = (torch.arange(-7, 7) + 0.5 if symmetric else torch.arange(0, 14) + 0.5) * s
        up, down = (torch.nextafter(half, torch.full_like(half, d)) for d in (torch.inf, -torch.inf))
        near = half * (1 + (torch.rand(64 - 42 - 1, 14, generator=g)[0] - 0.5) * 2.0 ** -14)
        w = torch.cat((top, half, up, down, near))
        rows.append(torch.nn.functional.pad(w, (0, 64 - len(w))))
    w = torch.stack(rows)
    got = gh.quantize_grouped_i4(w.to(torch_dev), 64, symmetric=symmetric)
    for a, b in zip(got, W.quantize(w, 64, symmetric)):
        assert (a is None) == (b is None) and (a is None or torch.equal(a.cpu(), b))


def test_quantize_borders_and_nan(torch_dev):
    gh = _gh()
    w = torch.zeros(4, 32)
    w[0] = torch.arange(32) * 0.5 - 7.0        # ties between two codes, clamped above
    w[0, 31] = 7.0
    w[1, 3] = float("nan")
    w[1, 4] = 3.5
    w[2] = float("nan")
    w[3, 0] = 1e-45
    for symmetric in (True, False):
        got = gh.quantize_grouped_i4(w.to(torch_dev), 32, symmetric=symmetric)
        clean = w.nan_to_num(0.0)
        want = W.quantize(clean, 32, symmetric)
        assert torch.equal(got[0][:3].cpu(), want[0][:3]) and torch.equal(got[1][:3].cpu(), want[1][:3])
        assert torch.isfinite(got[1]).all() and (got[1] > 0).all()


def _linear(dev, x, wt, group, bias=None, **kw):
    gh = _gh()
    d = lambda t: None if t is None else t.to(dev)  # noqa: E731
    y = gh.linear_w4(d(x), d(wt[0]), d(wt[1]), d(wt[2]), d(bias), group_size=group, **kw)
    torch.cuda.synchronize()
    return y.cpu()


SHAPES = [(1, 1, 32, 32), (2, 5, 64, 32), (3, 40, 1024, 128), (4, 4100, 96, 32), (1, 3000, 4096, 128),
          (5, 33, 256, 64), (16, 100, 416, 32), (17, 64, 1024, 128), (33, 200, 800, 128), (50, 130, 2048, 64),
          (64, 65, 544, 256), (80, 70, 320, 96), (6, 20, 20000 // 32 * 32, 128), (1, 9, 14336, 128),
          (9, 700, 352, 1024), (130, 300, 288, 32)]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda v: "x".join(map(str, v)))
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("zeros", [False, True])
def test_linear_whole_numbers_are_exact(torch_dev, shape, kind, zeros):
    """Whole x, scales that are powers of two: every sum is exact in fp32, so
    the result is the 64-bit one rounded once."""
    m, n, k, group = shape
    g = torch.Generator().manual_seed(m * n + k)
    wt = W.random_weight(n, k, group, zeros, seed=k + n, exact=True)
    x = torch.randint(-3, 4, (m, k), generator=g).to(W.TYPES[kind])
    bias = torch.randint(-9, 10, (n,), generator=g).to(W.TYPES[kind])
    want = x.double() @ W.weight(*wt, group).t() + bias.double()
    assert torch.equal(_linear(torch_dev, x, wt, group, bias), want.to(W.TYPES[kind]))


@pytest.mark.parametrize("shape", SHAPES, ids=lambda v: "x".join(map(str, v)))
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_linear_random(torch_dev, shape, kind):
    """Sums of k fp32 products in any order: each of the at most k roundings of
    a sum, and two more per product, is 2^-24 of no more than the sum of
    magnitudes; one rounding to the output's type."""
    m, n, k, group = shape
    g = torch.Generator().manual_seed(m + n + k)
    wt = W.random_weight(n, k, group, True, seed=k)
    x = torch.randn(m, k, generator=g).to(W.TYPES[kind])
    w = W.weight(*wt, group)
    want = x.double() @ w.t()
    size = x.double().abs() @ w.abs().t()
    bound = (k + 2) * 2.0 ** -24 * size + torch.finfo(W.TYPES[kind]).eps / 2 * (want.abs() * (1 + 2 ** -9))
    assert (_linear(torch_dev, x, wt, group).double() - want).abs().le(bound).all()


# up to 16 rows: ragged slices, row blocks and groups, a group longer than the
# rows, and scales that fill the table (8192 columns in groups of 32)
FEW = [(3, 17, 96, 32), (5, 16, 128, 128), (16, 100, 160, 96), (9, 33, 4128, 64), (16, 40, 8192, 32), (4, 24, 992, 1024),
       (12, 48, 1280, 160), (16, 16, 544, 192), (7, 1, 32, 32), (13, 31, 2080, 256)]


@pytest.mark.parametrize("shape", FEW, ids=lambda v: "x".join(map(str, v)))
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("zeros", [False, True])
def test_linear_few_rows(torch_dev, shape, kind, zeros):
    """As above: exact sums of whole numbers, then random ones."""
    m, n, k, group = shape
    g = torch.Generator().manual_seed(m * n + k + 1)
    wt = W.random_weight(n, k, group, zeros, seed=k + n, exact=True)
    x = torch.randint(-3, 4, (m, k), generator=g).to(W.TYPES[kind])
    want = x.double() @ W.weight(*wt, group).t()
    assert torch.equal(_linear(torch_dev, x, wt, group), want.to(W.TYPES[kind]))
    wt = W.random_weight(n, k, group, zeros, seed=k)
    x = torch.randn(m, k, generator=g).to(W.TYPES[kind])
    w = W.weight(*wt, group)
    want, size = x.double() @ w.t(), x.double().abs() @ w.abs().t()
    if kind == "bf16":  # sums of c x and of z x, up to 15 |x| s each
        size = size + 15 * x.double().abs() @ torch.ones_like(w).t() * w.abs().max()
    bound = (k + 4) * 2.0 ** -24 * size + torch.finfo(W.TYPES[kind]).eps / 2 * (want.abs() * (1 + 2 ** -9))
    assert (_linear(torch_dev, x, wt, group).double() - want).abs().le(bound).all()


@pytest.mark.parametrize("m", [2, 3, 7, 17])
def test_linear_rows_far_apart(torch_dev, m):
    """Rows of x whose distances pass 32 bits, in elements and in bytes."""
    gh = _gh()
    k, n, group, ld = 288, 40, 64, 1 << 28
    wt = [t.to(torch_dev) for t in W.random_weight(n, k, group, True, seed=2)]
    rows = torch.randn(m, k, generator=torch.Generator().manual_seed(m)).to(torch_dev, torch.bfloat16)
    wide = torch.empty((m - 1) * ld + k, dtype=torch.bfloat16, device=torch_dev)
    x = wide.as_strided((m, k), (ld, 1))
    x.copy_(rows)
    a, b = gh.linear_w4(x, *wt, group_size=group), gh.linear_w4(rows, *wt, group_size=group)
    size = rows.double().cpu().abs() @ W.weight(*[t.cpu() for t in wt], group).abs().t()
    assert ((a.double() - b.double()).abs().cpu() <= 2.0 ** -8 * b.double().abs().cpu() + 32 * (k + 4) * 2.0 ** -24 * size).all()


@pytest.mark.parametrize("m", [2, 5, 16])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("group,zeros", [(128, False), (96, True)])
def test_linear_few_rows_of_a_large_weight(torch_dev, m, kind, group, zeros):
    """Of 2^27 codes and more, checked at some of its rows."""
    gh = _gh()
    n, k = 32769, 4096
    g = torch.Generator().manual_seed(m)
    codes, scales, zps = W.random_weight(64, k, group, zeros, seed=m)
    rows = torch.cat((torch.arange(16), torch.randint(0, n, (32,), generator=g), torch.arange(n - 16, n)))
    dev = [None if t is None else torch.zeros((n, t.shape[1]), dtype=t.dtype, device=torch_dev)
           for t in (codes, scales, zps)]
    for t, part in zip(dev, (codes, scales, zps)):
        if t is not None:
            t[rows.to(torch_dev)] = part.to(torch_dev)
    part = [None if t is None else t[rows.to(torch_dev)].cpu() for t in dev]  # (a row may be drawn twice)
    x = torch.randn(m, k, generator=g).to(W.TYPES[kind])
    got = gh.linear_w4(x.to(torch_dev), *dev, group_size=group).double().cpu()[:, rows]
    w = W.weight(*part, group)
    want, size = x.double() @ w.t(), x.double().abs() @ w.abs().t()
    bound = (k + 2) * 2.0 ** -24 * size + torch.finfo(W.TYPES[kind]).eps / 2 * (want.abs() * (1 + 2 ** -9))
    assert (got - want).abs().le(bound).all()


@pytest.mark.parametrize("m", [1, 3, 16, 17, 64])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("zeros", [False, True])
def test_linear_workspace_of_the_asked_size(torch_dev, m, kind, zeros):
    """The size is asked for without the zero points and the strides, and is
    enough with and without them."""
    gh = _gh()
    for n, k, group in ((80, 4096, 32), (80, 16384, 32), (300, 8192, 128)):
        wt = W.random_weight(n, k, group, zeros, seed=k)
        x = torch.randn(m, k, generator=torch.Generator().manual_seed(m)).to(W.TYPES[kind])
        size = gh.linear_w4_workspace_size(m, n, k, group, W.TYPES[kind])
        ws = torch.empty(max(size, 16), dtype=torch.uint8, device=torch_dev)
        dev = [None if t is None else t.to(torch_dev) for t in wt]
        got = gh.linear_w4(x.to(torch_dev), *dev, group_size=group, workspace=ws)
        assert torch.equal(got.cpu(), _linear(torch_dev, x, wt, group))


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_linear_rows_of_zeros_give_zeros(torch_dev, kind):
    """A weight row whose codes are all its zero point adds nothing, not even a
    rounding, whatever x is."""
    k, n, group = 2048, 20, 128
    x = (torch.randn(8, k, generator=torch.Generator().manual_seed(9)) * 1e3).to(W.TYPES[kind])
    wt = list(W.random_weight(n, k, group, False, seed=8))
    wt[0][3] = 0x88
    y = _linear(torch_dev, x, wt, group)
    assert (y[:, 3] == 0).all() and not (y == 0).all(0)[:3].any()


@pytest.mark.parametrize("m", [1, 4, 7, 40])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_linear_rows_of_very_different_size(torch_dev, m, kind):
    """Rows, and slices of a row, that lie powers of two apart keep their own
    relative accuracy (relative to their own magnitudes)."""
    k, n, group = 1024, 48, 64
    g = torch.Generator().manual_seed(m)
    wt = W.random_weight(n, k, group, True, seed=3)
    x = torch.randn(m, k, generator=g)
    x *= 2.0 ** torch.linspace(-100, 90, m).round()[:, None]
    x = x.to(W.TYPES[kind])
    w = W.weight(*wt, group)
    want = x.double() @ w.t()
    size = x.double().abs() @ w.abs().t()
    bound = (k + 2) * 2.0 ** -24 * size + torch.finfo(W.TYPES[kind]).eps / 2 * want.abs() * (1 + 2 ** -9)
    assert (_linear(torch_dev, x, wt, group).double() - want).abs().le(bound).all()


@pytest.mark.parametrize("m", [1, 3, 6, 50])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
def test_linear_values_that_are_not_finite_stay_in_their_row(torch_dev, m, kind, value):
    k, n, group = 512, 40, 128
    g = torch.Generator().manual_seed(m)
    wt = W.random_weight(n, k, group, False, seed=4)
    x = torch.randn(m, k, generator=g).to(W.TYPES[kind])
    ref = _linear(torch_dev, x, wt, group)
    x[m - 1, 77] = value
    got = _linear(torch_dev, x, wt, group)
    assert torch.equal(got[:m - 1], ref[:m - 1])
    c = W.unpack(wt[0])[:, 77].int() - 8
    if value != value:
        assert torch.isnan(got[m - 1]).all()
    else:
        assert torch.isinf(got[m - 1][c > 0]).all() and (got[m - 1][c > 0] > 0).all()
        assert (got[m - 1][c < 0] < 0).all() and torch.isnan(got[m - 1][c == 0]).all()


@pytest.mark.parametrize("m", [1, 20])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_linear_strided_rows_and_out(torch_dev, m, kind):
    gh = _gh()
    k, n, group = 640, 50, 32
    wt = [None if t is None else t.to(torch_dev) for t in W.random_weight(n, k, group, True, seed=5)]
    wide = torch.randn(m, k + 37, device=torch_dev).to(W.TYPES[kind])
    for at in (0, 1, 8, 37):  # 16-byte aligned rows and others
        x = wide[:, at:at + k]
        want = gh.linear_w4(x.contiguous(), *wt, group_size=group)
        out = torch.empty_like(want)
        assert gh.linear_w4(x, *wt, group_size=group, out=out) is out
        assert torch.equal(out, want)


def test_linear_on_a_quantized_weight(torch_dev):
    """quantize -> Linear is Linear on the dequantized weight."""
    gh = _gh()
    g = torch.Generator().manual_seed(6)
    w = (torch.randn(300, 1088, generator=g) * 0.02).to(torch_dev)
    for symmetric in (True, False):
        q = gh.quantize_grouped_i4(w, 64, symmetric=symmetric)
        back = gh.dequantize_grouped_i4(*q, 64).double().cpu()
        for m in (1, 30):
            x = torch.randn(m, 1088, generator=g)
            y = gh.linear_w4(x.to(torch_dev), *q, group_size=64).double().cpu()
            size = x.double().abs() @ back.abs().t()
            assert (y - x.double() @ back.t()).abs().le(1091 * 2.0 ** -24 * size).all()


def test_captured_linear_replays(torch_dev):
    gh = _gh()
    k, n, group = 4096, 512, 128
    wt = [None if t is None else t.to(torch_dev) for t in W.random_weight(n, k, group, True, seed=7)]
    x = torch.randn(16, k, device=torch_dev)
    y = torch.empty(16, n, device=torch_dev)
    size = gh.linear_w4_workspace_size(16, n, k)
    assert size > 0
    ws = torch.empty(size, dtype=torch.uint8, device=torch_dev)
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(g, stream=s):
        gh.linear_w4(x, *wt, group_size=group, out=y, workspace=ws)
    for rep in range(4):
        x.normal_()
        ws.fill_(0xff)
        want = gh.linear_w4(x, *wt, group_size=group)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want), rep


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("k,group,n", [(2100384, 2097184, 32), (8388608, 786336, 5), (4194304, 1301664, 7)])
def test_linear_few_rows_in_very_long_groups(torch_dev, kind, k, group, n):
    """x is not zero at the ends of the groups only, whole there, and scales are
    powers of two: exact."""
    gh = _gh()
    m = 4
    g = torch.Generator().manual_seed(k)
    at = torch.arange(k)
    at = at[(at % group >= group - 96) | (at % group < 64) | (at >= k - 64)]
    codes = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, generator=g)
    groups = -(-k // group)
    scales = 2.0 ** (torch.arange(groups) % 8 - 4).float()[None] * 2.0 ** torch.randint(0, 2, (n, 1), generator=g)
    zps = torch.randint(0, 16, (n, groups), dtype=torch.uint8, generator=g)
    x = torch.zeros(m, k)
    x[:, at] = torch.randint(-1, 2, (m, len(at)), generator=g).float()
    c = (codes[:, at // 2] >> (at % 2 * 4).to(torch.uint8)) & 15
    w = (c.double() - zps[:, at // group].double()) * scales[:, at // group].double()
    got = gh.linear_w4(x.to(W.TYPES[kind]).to(torch_dev), codes.to(torch_dev), scales.to(torch_dev), zps.to(torch_dev),
                       group_size=group)
    assert torch.equal(got.cpu(), (x[:, at].double() @ w.t()).to(W.TYPES[kind]))


@pytest.mark.parametrize("m", [3, 5, 16, 40])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("zeros", [False, True])
def test_linear_many_groups_and_values_far_below_the_largest(torch_dev, m, kind, zeros):
    """448 groups to a row, 3 to 16 rows among them.  Every 256th column of x is 1
    and meets a weight of 0, the others are some 2^-20 (f16: 2^-12) of it: the result
    is theirs alone.  Each may lose 2^-39 of the 1 (half the last bit of an f16
    subnormal after the scaling, which f16 itself has not); then sums."""
    n, k, group = 40, 14336, 32
    g = torch.Generator().manual_seed(m)
    wt = W.random_weight(n, k, group, zeros, seed=m + 60)
    z = 8 if wt[2] is None else wt[2][:, ::256 // group]
    wt[0][:, ::128] = wt[0][:, ::128] & 0xf0 | z
    x = (torch.randn(m, k, generator=g) * (2.0 ** -12 if kind == "f16" else 2.0 ** -20)).to(W.TYPES[kind])
    x[:, ::256] = 1
    w = W.weight(*wt, group)
    assert (w[:, ::256] == 0).all()
    want, small = x.double() @ w.t(), x.double().abs() @ w.abs().t()
    lost = 0.0 if kind == "f16" else 2.0 ** -39 * w.abs().sum(1)
    bound = (k + 4) * 2.0 ** -24 * small + lost + torch.finfo(W.TYPES[kind]).eps / 2 * want.abs() * (1 + 2 ** -9)
    if kind == "f16":
        bound = bound + 2.0 ** -25  # (the result may be subnormal)
    assert (_linear(torch_dev, x, wt, group).double() - want).abs().le(bound).all()


@pytest.mark.parametrize("shape", FEW, ids=lambda v: "x".join(map(str, v)))
@pytest.mark.parametrize("zeros", [False, True])
def test_linear_few_rows_of_bf16_by_group(torch_dev, shape, zeros):
    """x in one group at a time, so that a lost group or another's scale shows: sums
    of c x and of z x are off by (terms + 4) 2^-24 of the sum of (c + z) |x| s at most,
    then one rounding to the type."""
    m, n, k, group = shape
    g = torch.Generator().manual_seed(m * n + k + 2)
    wt = W.random_weight(n, k, group, zeros, seed=k + 70)
    x = torch.randn(m, k, generator=g).to(torch.bfloat16)
    w = W.weight(*wt, group)
    z = 8.0 if wt[2] is None else W.spread(wt[2], k, group).double()
    both = (W.unpack(wt[0]).double() + z) * W.spread(wt[1], k, group).double()
    groups = -(-k // group)
    for at in sorted({0, groups // 2, groups - 1, int(torch.randint(0, groups, (1,), generator=g))}):
        cut = slice(at * group, min(k, at * group + group))
        part = torch.zeros_like(x)
        part[:, cut] = x[:, cut]
        want = part.double() @ w.t()
        size = part.double().abs() @ both.t()
        bound = (cut.stop - cut.start + 4) * 2.0 ** -24 * size + 2.0 ** -8 * want.abs() * (1 + 2 ** -9)
        assert (_linear(torch_dev, part, wt, group).double() - want).abs().le(bound).all(), at
    want, size = x.double() @ w.t(), x.double().abs() @ both.t()
    bound = (k + 4) * 2.0 ** -24 * size + 2.0 ** -8 * want.abs() * (1 + 2 ** -9)
    assert (_linear(torch_dev, x, wt, group).double() - want).abs().le(bound).all()
