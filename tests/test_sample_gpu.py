"""Sampling on the GPU against its definition in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
INF, NAN = float("inf"), float("nan")


def _gh():
    import ghostflow_hip as gh

    return gh


def plain(x, u, t, k, p, least):
    """(tokens that may be drawn, logarithm of each one's probability): one, or two
    where u is within 2^-32 of the border between them (weights are held to 2^-45 of
    the largest, up to 2^13 times the root of 2^19 of them off in their sum)."""
    x = x.double()
    x = torch.where(x.isnan(), -INF, x)
    top = x.max()
    if top == -INF:
        return {-1: NAN}
    best = int(torch.nonzero(x == top)[0])
    if not t > 0:
        return {best: 0.0}
    z = torch.where(x == top, 0.0, (x - top) / t)
    w = torch.where((x == -INF) | z.isnan(), 0.0, torch.exp(z))
    order = torch.sort(x, descending=True, stable=True).indices
    s = w[order]
    n = k if 0 < k < len(x) else len(x)
    if p < 1:
        before = torch.cumsum(s[:n], 0) - s[:n]
        n = max(1, int((before < p * s[:n].sum()).sum()))
    if least > 0:
        n = max(1, int((s[:n] >= least).sum()))
    keep = order[:n].sort().values
    c = torch.cumsum(w[keep], 0)
    total = float(c[-1])
    at = u * total
    out = {}
    for d in (-2.0 ** -32, 0.0, 2.0 ** -32):
        i = int(torch.searchsorted(c, torch.tensor([min(max(at + d * total, 0.0), total * (1 - 2.0 ** -50))],
                                                   dtype=torch.float64), right=True)[0])
        i = min(i, len(keep) - 1)
        out[int(keep[i])] = float(z[keep[i]]) - math.log(total)
    return out


def check(x, u, t, k, p, least, *, dev, **kw):
    """Tensors of settings on the CPU, one per row; x on any device."""
    got, lp = _gh().sample(x.to(dev) if x.device != dev else x, u.to(dev), temperature=t.to(dev), top_k=k.to(dev),
                           top_p=p.to(dev), min_p=least.to(dev), want_logprobs=True, **kw)
    x = x.cpu()
    for r in range(len(x)):
        want = plain(x[r], float(u[r]), float(t[r]), int(k[r]), float(p[r]), float(least[r]))
        token = int(got[r])
        assert token in want, (r, token, want, float(t[r]), int(k[r]), float(p[r]), float(least[r]), float(u[r]))
        a, b = float(lp[r]), want[token]
        # one rounding to fp32 of a number good to 2^-32
        assert (math.isnan(a) and math.isnan(b)) or abs(a - b) <= 2.0 ** -24 * abs(b) + 2.0 ** -30, (r, a, b)
    return got


# temperature, top_k, top_p, min_p
SETTINGS = [
    (1.0, 0, 1.0, 0.0), (0.7, 50, 0.9, 0.0), (0.0, 0, 1.0, 0.0), (1.3, 0, 0.95, 0.0), (0.6, 0, 0.5, 0.0), (1.0, 0, 1.0, 0.1),
    (1.0, 1, 1.0, 0.0), (2.0, 300, 1.0, 0.0), (1.0, 2000, 0.99, 0.0), (1.0, 3000, 1.0, 0.0), (1.5, 3000, 0.8, 0.01),
    (1.0, 0, 0.999, 0.001), (3.0, 0, 0.9999, 0.0), (1.0, 0, 1.0, 1e-6), (0.05, 0, 1.0, 0.0), (INF, 0, 1.0, 0.0),
    (INF, 7, 0.5, 0.0), (1.0, 10 ** 9, 2.0, -1.0), (1.0, 0, 0.0, 0.0), (1.0, 40, 1.0, 1.0), (-1.0, 5, 0.5, 0.5),
    (1e-30, 0, 0.9, 0.0), (100.0, 0, 0.3, 0.0), (1.0, 0, -0.5, 0.2),
]


def settings(rows=None):
    rows = rows or len(SETTINGS)
    t, k, p, least = zip(*(SETTINGS[i % len(SETTINGS)] for i in range(rows)))
    f = lambda v: torch.tensor(v, dtype=torch.float32)  # noqa: E731
    return f(t), torch.tensor(k, dtype=torch.int32), f(p), f(least)


def logits(rows, vocab, kind, g, std=2.0, peaks=20):
    x = torch.randn(rows, vocab, generator=g) * std
    x += 8.0 * (torch.rand(rows, vocab, generator=g) < peaks / vocab)
    return x.to(TYPES[kind])


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("vocab", [1, 2, 15, 16, 17, 100, 1000, 4095, 4097, 5000, 32000, 50257])
def test_settings(torch_dev, kind, vocab):
    g = torch.Generator().manual_seed(vocab)
    x = logits(len(SETTINGS), vocab, kind, g)
    for _ in range(2):
        check(x, torch.rand(len(x), generator=g), *settings(), dev=torch_dev)


@pytest.mark.parametrize("kind,vocab", [("bf16", 131072), ("f32", 2 ** 19), ("f16", 2 ** 19 - 5)])
def test_large_vocabularies(torch_dev, kind, vocab):
    g = torch.Generator().manual_seed(vocab)
    x = logits(len(SETTINGS), vocab, kind, g)
    check(x, torch.rand(len(x), generator=g), *settings(), dev=torch_dev)


@pytest.mark.parametrize("vocab", [7, 1000, 9001, 70000])
def test_equal_logits(torch_dev, vocab):
    """Cuts inside runs of equal logits go by the index, and fall where the weights'
    exact sums have them."""
    g = torch.Generator().manual_seed(vocab)
    for x in (torch.zeros(len(SETTINGS), vocab), torch.randint(-2, 2, (len(SETTINGS), vocab), generator=g).float(),
              torch.randint(0, 2, (len(SETTINGS), vocab), generator=g).float() * -0.0):
        check(x, torch.rand(len(x), generator=g), *settings(), dev=torch_dev)
    # a half, a quarter of equal ones: 0.5 and 0.25 of n sum to whole weights
    n = vocab - vocab % 4 or 4
    x = torch.zeros(4, max(n, 4))
    t, k, p, least = (torch.tensor(v) for v in ([1.0] * 4, [0, 0, n // 2, 0], [0.5, 0.25, 0.5, 0.75], [0.0] * 4))
    got = _gh().sample(x.to(torch_dev), torch.full((4,), 1 - 2.0 ** -24, device=torch_dev), temperature=t.to(torch_dev),
                       top_k=k.int().to(torch_dev), top_p=p.to(torch_dev))
    assert got.tolist() == [n // 2 - 1, n // 4 - 1, n // 4 - 1 + (n // 2 % 2), 3 * n // 4 - 1]


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_parts_of_a_row_on_different_levels(torch_dev, kind):
    """Runs of 4096 logits whose largest lie from nothing to far apart, the cut among
    a few values or many, around 0 and away from it."""
    g = torch.Generator().manual_seed(11)
    n = 60
    t = torch.tensor([0.3, 1.0, 1.7, 6.0]).repeat(n // 4)
    p = torch.rand(n, generator=g) * 0.98 + 0.01
    least = torch.where(torch.arange(n) % 5 == 4, 0.02, 0.0)
    k = torch.where(torch.arange(n) % 7 == 6, 500, 0).int()
    levels = torch.tensor([-100.0, -21.0, -5.0, -1.9, -0.5, -0.06, 0.0, 0.0])
    for spread in (0.02, 1.0, 8.0):
        x = torch.rand(n, 30000, generator=g) * spread
        x += levels[torch.randint(0, 8, (n, 8), generator=g)].repeat_interleave(4096, 1)[:, :30000]
        x += torch.tensor([0.0, -spread / 2, 40.0])[torch.arange(n) % 3, None]
        check(x.to(TYPES[kind]), torch.rand(n, generator=g), t, k, p, least, dev=torch_dev)


def test_min_p_above_one(torch_dev):
    """No weight reaches it, so the first of the largest alone stays, however many are equal."""
    for vocab in (40, 3000, 9001, 70000):
        x = torch.zeros(3, vocab)
        x[0, 7:] = 2.0
        x[1, 1::2] = 0.5
        got = _gh().sample(x.to(torch_dev), torch.tensor([0.0, 0.5, 0.999], device=torch_dev), min_p=1.5)
        assert got.tolist() == [7, 1, 0], vocab


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("vocab,k", [(600, 555), (1644, 1100), (4096, 2500), (7168, 7000), (7169, 4096), (40000, 1500),
                                     (131072, 4000)])
def test_many_candidates(torch_dev, kind, vocab, k):
    """More than are put in order, up to all that can be listed, and past that; equal
    logits at the cut, all in a narrow range, and of very different size."""
    g = torch.Generator().manual_seed(vocab)
    x = torch.cat([torch.randn(4, vocab, generator=g), torch.randn(2, vocab, generator=g) * 1e-3,
                   torch.randint(-3, 3, (2, vocab), generator=g).float(), torch.randn(2, vocab, generator=g) * 1e3,
                   torch.randn(2, vocab, generator=g) - 50.0])
    n = len(x)
    t = torch.tensor([1.0, 2.0, 0.7]).repeat(n // 3)
    p = torch.tensor([1.0, 0.9, 0.5, 0.999]).repeat(n // 4)
    least = torch.where(torch.arange(n) % 3 == 2, 0.004, 0.0)
    for ks in (torch.full((n,), k), torch.where(torch.arange(n) % 2 == 0, 0, k // 2)):
        check(x.to(TYPES[kind]), torch.rand(n, generator=g), t, ks.int(), p, least, dev=torch_dev)


def test_infinite_and_nan_logits(torch_dev):
    for vocab in (40, 6000):
        g = torch.Generator().manual_seed(vocab)
        x = logits(len(SETTINGS), vocab, "f32", g)
        x[:, ::3] = -INF
        x[:, 1::7] = NAN
        check(x, torch.rand(len(x), generator=g), *settings(), dev=torch_dev)
        x[:, 5] = INF
        x[:, vocab - 4] = INF
        x[3:, 20] = INF
        check(x, torch.rand(len(x), generator=g), *settings(), dev=torch_dev)
        x[:] = -INF
        x[::2, vocab // 2] = -3e38
        x[1::4] = NAN
        got = check(x, torch.rand(len(x), generator=g), *settings(), dev=torch_dev)
        assert (got[::2] == vocab // 2).all() and (got[1::2] == -1).all()
        x = torch.full((len(SETTINGS), vocab), 3.4e38)
        x[:, ::2] = -3.4e38
        check(x, torch.rand(len(x), generator=g), *settings(), dev=torch_dev)


@pytest.mark.parametrize("vocab", [700, 3000, 7000])
def test_infinite_and_nan_among_many_candidates(torch_dev, vocab):
    g = torch.Generator().manual_seed(vocab)
    for filled in (0.3, 0.95):
        x = logits(len(SETTINGS), vocab, "f32", g)
        x[torch.rand(x.shape, generator=g) < filled] = -INF
        x[torch.rand(x.shape, generator=g) < 0.05] = NAN
        check(x, torch.rand(len(x), generator=g), *settings(), dev=torch_dev)
        x[:, 11] = -3e38
        x[::2, 600:620] = INF
        check(x, torch.rand(len(x), generator=g), *settings(), dev=torch_dev)
        check(x * 1e-38, torch.rand(len(x), generator=g), *settings(), dev=torch_dev)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_rows_that_begin_anywhere(torch_dev, kind):
    g = torch.Generator().manual_seed(3)
    whole = logits(len(SETTINGS), 5003, kind, g).to(torch_dev)
    u = torch.rand(len(SETTINGS), generator=g)
    for x in (whole[:, 1:], whole[:, 3:4990], whole[:, :7]):
        check(x, u, *settings(), dev=torch_dev)


def test_first_and_last_numbers(torch_dev):
    """u = 0 draws the first that is left, the largest below 1 (and what is not below
    it) the last."""
    x = torch.tensor([[-INF, 1.0, 2.0, -INF, 0.0, -50.0, -INF]] * 5)
    u = torch.tensor([0.0, 1 - 2.0 ** -24, 1.0, 7.0, -3.0])
    got = _gh().sample(x.to(torch_dev), u.to(torch_dev))
    # (e^-52 = 2^-75 is no weight any more, and less than the last step of u)
    assert got.tolist() == [1, 4, 4, 4, 1]
    got = _gh().sample(x.to(torch_dev), u.to(torch_dev), top_k=3, min_p=0.2)
    assert got.tolist() == [1, 2, 2, 2, 1]


@pytest.mark.parametrize("filters", [{}, {"top_k": 60}, {"top_p": 0.8}, {"min_p": 0.02, "temperature": 1.5}])
def test_frequencies(torch_dev, filters):
    """With u at the middles of 4000 equal steps a token comes up as often as its
    probability says, to within one."""
    g = torch.Generator().manual_seed(5)
    n, vocab = 4000, 300
    x = torch.randn(vocab, generator=g) * 2
    u = (torch.arange(n) + 0.5) / n
    got = _gh().sample(x.to(torch_dev).expand(n, vocab).contiguous(), u.to(torch_dev), **filters).cpu()
    z = x.double() / filters.get("temperature", 1.0)
    w = torch.exp(z - z.max())
    order = torch.sort(w, descending=True).indices
    if "top_k" in filters:
        w[order[filters["top_k"]:]] = 0
    if "top_p" in filters:
        before = torch.cumsum(w[order], 0) - w[order]
        w[order[before >= torch.tensor(filters["top_p"]).double() * w.sum()]] = 0
    if "min_p" in filters:
        w[w < filters["min_p"]] = 0
    assert ((torch.bincount(got.long(), minlength=vocab) - n * w / w.sum()).abs() <= 1).all()
    assert torch.equal(got, got.sort().values)


def test_numbers_for_settings(torch_dev):
    """One number for all rows is a tensor of it."""
    g = torch.Generator().manual_seed(6)
    x, u = logits(9, 700, "f32", g).to(torch_dev), torch.rand(9, generator=g).to(torch_dev)
    full = lambda v: torch.full((9,), v, device=torch_dev)  # noqa: E731
    for t, k, p, m in SETTINGS:
        a = _gh().sample(x, u, temperature=t, top_k=k, top_p=p, min_p=m, want_logprobs=True)
        b = _gh().sample(x, u, temperature=full(t), top_k=full(k).int(), top_p=full(p), min_p=full(m), want_logprobs=True)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    out = torch.full((9,), -7, dtype=torch.int32, device=torch_dev)
    assert _gh().sample(x, u, top_k=2 ** 40, out=out) is out and (out >= 0).all()
    assert torch.equal(out, _gh().sample(x, u))
    assert _gh().sample(x[:0], u[:0]).shape == (0,)


def test_captured_and_on_streams(torch_dev):
    """A graph replayed with other logits, numbers and settings, eager calls between;
    two streams at once."""
    gh = _gh()
    g = torch.Generator().manual_seed(7)
    n = len(SETTINGS)
    x = logits(n, 20000, "bf16", g).to(torch_dev)
    u = torch.rand(n, generator=g).to(torch_dev)
    now = dict(zip(("temperature", "top_k", "top_p", "min_p"), (t.to(torch_dev) for t in settings())))
    out = torch.zeros(n, dtype=torch.int32, device=torch_dev)
    ws = torch.full((gh.sample_workspace_size(n, 20000),), 255, dtype=torch.uint8, device=torch_dev)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        gh.sample(x, u, out=out, workspace=ws, **now)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        gh.sample(x, u, out=out, workspace=ws, **now)
    for i in range(4):
        x.copy_(logits(n, 20000, "bf16", g))
        u.copy_(torch.rand(n, generator=g))
        for t in now.values():
            t.copy_(t.roll(1))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, gh.sample(x, u, **now))
        torch.cuda.synchronize()
    other = torch.cuda.Stream()
    y = logits(n, 9000, "f32", g).to(torch_dev)
    want = gh.sample(x, u, **now), gh.sample(y, u, **now)
    torch.cuda.synchronize()
    a, b = [], []
    for _ in range(4):
        with torch.cuda.stream(s):
            a.append(gh.sample(x, u, **now))
        with torch.cuda.stream(other):
            b.append(gh.sample(y, u, **now))
    torch.cuda.synchronize()
    assert all(torch.equal(t, want[0]) for t in a) and all(torch.equal(t, want[1]) for t in b)


def test_many_rows(torch_dev):
    g = torch.Generator().manual_seed(8)
    x = logits(3000, 50, "f16", g)
    check(x, torch.rand(3000, generator=g), *settings(3000), dev=torch_dev)


def test_a_step_from_hidden_states_to_tokens(torch_dev):
    """The run of a step: norms, 8-bit cache, attention, the head's projection and
    a token, the same twice, and the token that the logits have by the definition."""
    gh = _gh()
    torch.manual_seed(9)
    e, heads, vocab = 128, 4, 900
    m = gh.MultiHeadAttention(e, heads)
    m.eval()
    m.enable_qk_norm()
    head = gh.GroupQuantizedLinear((torch.randn(vocab, e) * 0.3).to(torch_dev), None, group_size=32)
    x, u = (torch.randn(21, e) * 0.5).to(torch_dev), torch.rand(3)
    tokens = []
    for _ in range(2):
        c = gh.PagedKVCache(8, 8, heads, e // heads, dtype=torch.uint8)
        ids = [c.add() for _ in range(3)]
        m.step_paged(x[:18], c, c.extend(ids, [9, 8, 1]))
        y = head(m.step_paged(x[18:], c, c.extend(ids, [1, 1, 1])))
        tokens.append(check(y, u, torch.full((3,), 0.8), torch.full((3,), 40, dtype=torch.int32), torch.full((3,), 0.9),
                            torch.zeros(3), dev=torch_dev))
    assert torch.equal(*tokens)


def test_numbers_past_fp32(torch_dev):
    """Numbers that fp32 does not hold count as infinite, a k past int32 as none."""
    gh = _gh()
    g = torch.Generator().manual_seed(2)
    x, u = torch.randn(50, 300, generator=g).to(torch_dev), torch.rand(50, generator=g).to(torch_dev)
    for a, b in ((dict(temperature=1e300), dict(temperature=INF)), (dict(top_p=-1e300), dict(top_p=0.0)),
                 (dict(min_p=1e39), dict(top_k=1)), (dict(top_k=10 ** 30), dict())):
        assert torch.equal(gh.sample(x, u, **a), gh.sample(x, u, **b)), a
    with pytest.raises(gh.GhostFlowError):
        gh.sample(x, u, temperature=NAN)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("low", [-31.5, -40.0, -100.0, -600.0])
@pytest.mark.parametrize("filters", [{}, {"top_p": 0.97}, {"top_k": 700}, {"min_p": 1e-6}, {"top_k": 5000, "top_p": 0.9999}])
def test_what_weighs_nothing_is_not_drawn(torch_dev, kind, low, filters):
    """Weights are held to 2^-45 of the largest, and e^-31.5 is less: u = 0 draws the first token
    that has one, numbers up to 1 and above the last, past whole runs of 4096 that have none."""
    g = torch.Generator().manual_seed(31)
    vocab = 6 * 4096 - 100
    x = torch.full((5, vocab), low)
    x[:, 9000:14000] = torch.randn(5, 5000, generator=g).clamp(-2, 2)
    x[1, :] = low
    x[1, 13000] = 0.0   # one alone
    x[2, 20000] = 0.5   # and one behind two runs without any
    x[3, 4096] = 1.0
    x[4, :9000] = -INF
    x = x.to(TYPES[kind])
    z = x.double() - x.double().amax(1, keepdim=True)
    w = torch.exp(z)
    order = torch.sort(x.float(), dim=1, descending=True, stable=True).indices
    for r in range(len(x)):
        s = w[r, order[r]]
        n = filters.get("top_k", vocab)
        if "top_p" in filters:
            n = max(1, int((torch.cumsum(s[:n], 0) - s[:n] < torch.tensor(filters["top_p"]).double() * s[:n].sum()).sum()))
        w[r, order[r, n:]] = 0
    w[w < max(filters.get("min_p", 0.0), 2.0 ** -45)] = 0
    first = (w > 0).int().argmax(1)
    last = vocab - 1 - (w > 0).flip(1).int().argmax(1)
    for u, want in ((0.0, first), (-1.0, first), (1.0, last), (3.0, last)):
        got = _gh().sample(x.to(torch_dev), torch.full((5,), u, device=torch_dev), **filters)
        assert got.tolist() == want.tolist(), u
