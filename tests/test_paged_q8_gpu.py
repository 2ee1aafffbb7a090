"""A paged cache of 8 bits on the GPU: codes and steps as the rule has them,
values read back, and attention over them against 64 bits."""
import math

import pytest
import torch

import _paged as P
import _q8 as Q

pytestmark = pytest.mark.gpu


def _gh():
    import ghostflow_hip as gh

    return gh


# ---- append and read ---------------------------------------------------------------

def _append(b, dev, *, cos=None, sin=None, interleaved=False, q_norm=None, k_norm=None, eps=1e-6, status=None):
    gh = _gh()
    x = Q.to(b, dev)
    move = lambda t: None if t is None else t.to(dev)  # noqa: E731
    extra = Q.scales(x) if "k_scales" in b else {}
    q = gh.paged_append(*P.args(x), x["k"], x["v"], q=x["q"], cos=move(cos), sin=move(sin), interleaved=interleaved,
                        q_norm=move(q_norm), k_norm=move(k_norm), norm_eps=eps, status=status, **extra)
    return q, x


def _expected(b, *, cos=None, sin=None, interleaved=False, k_norm=None, eps=1e-6):
    """Pages and step bytes after the append."""
    pages = {n: b[n].clone() for n in ("k_pages", "v_pages", "k_scales", "v_scales")}
    for s in range(len(b["kv_lens"])):
        a, e = int(b["q_offsets"][s]), int(b["q_offsets"][s + 1])
        for t in range(a, e):
            p = int(b["kv_lens"][s]) - (e - t)
            at, row = int(b["page_table"][s, p // b["page"]]), p % b["page"]
            k = Q.turned(Q.normed(b["k"][t], k_norm, eps), p, cos, sin, interleaved)
            for n, x in (("k", k), ("v", b["v"][t].float())):
                pages[n + "_pages"][at, row], pages[n + "_scales"][at, :, row] = Q.quantise(x)
    return pages


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("heads,kv_heads,d,rot,interleaved,norm", [
    (4, 2, 64, 64, False, True), (8, 8, 128, 64, True, True), (5, 1, 80, 80, False, False), (6, 3, 48, 8, False, True),
    (3, 1, 16, 16, True, False), (7, 1, 112, 0, False, True), (2, 2, 96, 24, True, True), (32, 8, 128, 128, False, False),
])
def test_codes_and_steps(torch_dev, kind, heads, kv_heads, d, rot, interleaved, norm):
    """Every byte of the cache, written or not, is the rule's: the norm's sum is in
    64 bits and every later operation is one fp32 rounding, so there is nothing
    to allow for.  The queries are within their one rounding, and the norm's and
    the rotation's few in fp32."""
    g = torch.Generator().manual_seed(d)
    b = Q.batch([3, 1, 0, 20], [19, 1, 4, 20], kind=kind, heads=heads, kv_heads=kv_heads, d=d, page=7, pad=2, seed=d)
    b["k"] *= 1.5
    cos, sin = P.angles(28, rot) if rot else (None, None)
    w = [1 + 0.3 * torch.randn(d, generator=g) if norm else None for _ in range(2)]
    q, x = _append(b, torch_dev, cos=cos, sin=sin, interleaved=interleaved, q_norm=w[0], k_norm=w[1])
    want = _expected(b, cos=cos, sin=sin, interleaved=interleaved, k_norm=w[1])
    for n, t in want.items():
        assert torch.equal(x[n].cpu(), t), n
    off = b["q_offsets"].tolist()
    for s, n in enumerate(b["kv_lens"].tolist()):
        for t in range(off[s], off[s + 1]):
            y = b["q"][t].double()
            if norm:
                y = y / (y.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w[0].double()
            size = y.abs().amax()
            y = P.turned(y, n - (off[s + 1] - t), cos, sin, interleaved)
            assert ((q[t].cpu().double() - y).abs() <= P.half_step(b["q"].dtype) * y.abs() + 8 * 2.0 ** -24 * size).all()
    # read back: the cached values rounded once
    pages = (x["k_pages"], x["v_pages"], x["page_table"], x["kv_lens"].new_tensor([0, 19, 20, 24, 44]), x["kv_lens"])
    for dt in P.TYPES.values():
        got = _gh().paged_read(*pages, dtype=dt, **Q.scales(x))
        for y, n in zip(got, ("k", "v")):
            rows = torch.cat([P.rows_of({**b, n + "_pages": Q.values(want[n + "_pages"], want[n + "_scales"].transpose(1, 2))},
                                        s)[0 if n == "k" else 1] for s in range(4)])
            assert torch.equal(y.cpu(), rows.to(dt))


@pytest.mark.parametrize("types", P.PAIRS)
@pytest.mark.parametrize("d,rot,interleaved,which", [(64, 64, False, "qk"), (80, 40, True, "k"), (24, 8, False, "q"),
                                                     (128, 0, False, "qk"), (8, 8, True, "qk")])
def test_norms_into_other_caches(torch_dev, types, d, rot, interleaved, which):
    """Norms and rotation against 64 bits: one rounding to the type, and three
    operations for the norm and three for the rotation in fp32 on values that the
    pair's length bounds."""
    g = torch.Generator().manual_seed(d + 1)
    b = P.batch([2, 0, 9], [30, 5, 9], heads=6, kv_heads=2, d=d, page=5, types=types, pad=1, seed=d)
    cos, sin = P.angles(30, rot) if rot else (None, None)
    w = {x: 1 + 0.3 * torch.randn(d, generator=g) for x in which}
    x = P.to(b, torch_dev)
    move = lambda t: None if t is None else t.to(torch_dev)  # noqa: E731
    q = _gh().paged_append(*P.args(x), x["k"], x["v"], q=x["q"], cos=move(cos), sin=move(sin), interleaved=interleaved,
                           q_norm=move(w.get("q")), k_norm=move(w.get("k")), norm_eps=1e-5)
    off = b["q_offsets"].tolist()
    written = torch.zeros(b["k_pages"].shape[:2], dtype=torch.bool)
    for s, n in enumerate(b["kv_lens"].tolist()):
        for t in range(off[s], off[s + 1]):
            p = n - (off[s + 1] - t)
            at, row = int(b["page_table"][s, p // b["page"]]), p % b["page"]
            written[at, row] = True
            for name, got in (("q", q[t]), ("k", x["k_pages"][at, row])):
                y = b[name][t].double()
                if name in w:
                    y = y / (y.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w[name].double()
                size = y.abs().amax()
                y = P.turned(y, p, cos, sin, interleaved)
                h = P.half_step(got.dtype)
                assert ((got.cpu().double() - y).abs() <= h * y.abs() + 8 * 2.0 ** -24 * size).all(), (name, t)
            assert torch.equal(x["v_pages"][at, row].cpu(), b["v"][t].to(b["v_pages"].dtype))
    for n in ("k_pages", "v_pages"):  # nothing else is touched
        assert torch.equal(x[n].cpu()[~written].nan_to_num(7.0), b[n][~written].nan_to_num(7.0))
    got = _gh().paged_read(x["k_pages"], x["v_pages"], x["page_table"], x["q_offsets"], x["kv_lens"], tokens=12,
                           dtype=torch.float32)
    for t in range(11):
        s = 0 if t < 2 else 2
        p = int(b["kv_lens"][s]) - (off[s + 1] - t)
        at, row = int(b["page_table"][s, p // 5]), p % 5
        assert torch.equal(got[0][t], x["k_pages"][at, row].float()) and torch.equal(got[1][t], x["v_pages"][at, row].float())
    assert (got[0][11] == 0).all()


def test_values_at_the_ends(torch_dev):
    """Zeros, the smallest and largest steps, halves between two codes, values
    that no step holds: their codes, and the bit of status."""
    d, inf, nan = 16, float("inf"), float("nan")
    rows = torch.zeros(12, 1, d)
    rows[1] = torch.arange(d) * 2.0 ** -22 * 4  # halves of the smallest step
    rows[2, 0, 0], rows[2, 0, 1] = 127 * 9 * 2.0 ** -10, 4.5 * 9 * 2.0 ** -10
    rows[3] = -(torch.arange(d) + 0.5) * 2.0 ** -5
    rows[4] = 15240.0
    rows[5] = torch.linspace(-15240, 15240, d)
    rows[6, 0, 3] = 1e-40
    rows[7] = torch.tensor([127.0, 126.5] * 8) * (1 + 2.0 ** -23)
    b = Q.batch([12], [12], kind="f32", heads=1, kv_heads=1, d=d, page=16, seed=1)
    b["k"], b["v"] = rows, rows.flip(0)
    status = torch.zeros(1, dtype=torch.int32, device=torch_dev)
    _, x = _append(b, torch_dev, status=status)
    for n, t in _expected(b).items():
        assert torch.equal(x[n].cpu(), t), n
    assert int(status) == 0
    for bad in (inf, -inf, nan, 15240.0 * (1 + 2.0 ** -22), -3e38):
        rows[2, 0, 5] = bad
        b["k"], b["v"] = rows, torch.zeros_like(rows)
        status.zero_()
        _, x = _append(b, torch_dev, status=status)
        for n, t in _expected(b).items():
            assert torch.equal(x[n].cpu(), t), (bad, n)
        assert int(status) == 4, bad


def test_what_cannot_be_written(torch_dev):
    """Bad pages and lengths: nothing is written for them, their bits are set,
    reading gives zeros or leaves the row."""
    b = Q.batch([4, 4], [8, 8], kind="bf16", heads=2, kv_heads=2, d=32, page=4, seed=2)
    b["page_table"][0, 1] = -1
    b["page_table"][1, 1] = 10 ** 6
    status = torch.zeros(1, dtype=torch.int32, device=torch_dev)
    _, x = _append(b, torch_dev, status=status)
    for n in ("k_pages", "v_pages", "k_scales", "v_scales"):
        assert torch.equal(x[n].cpu(), b[n])
    assert int(status) == 2
    status.zero_()
    k, v = (torch.full((8, 2, 32), 5.0, device=torch_dev) for _ in range(2))
    _gh().paged_read(*P.args(x), k_out=k, v_out=v, status=status, **Q.scales(x))
    assert int(status) == 2 and (k == 0).all() and (v == 0).all()
    x["kv_lens"][0] = 2  # two of its four tokens lie before position 0
    x["kv_lens"][1] = 11  # the table holds 8
    x["page_table"].zero_()
    status.zero_()
    k.fill_(5.0)
    _gh().paged_read(*P.args(x), k_out=k, v_out=v, status=status, **Q.scales(x))
    assert int(status) == 1 and (k[:2] == 5).all() and (k[2:4] != 5).any() and (k[5:] == 5).all()


@pytest.mark.parametrize("cache,kind,kv_heads,d", [("u8", "bf16", 2, 64), ("u8", "f32", 1, 16), ("u8", "f16", 3, 80),
                                                   ("bf16", "f32", 2, 64), ("f16", "f16", 4, 128), ("f32", "bf16", 1, 24)])
@pytest.mark.parametrize("page", [16, 5])
def test_many_small_rows_read(torch_dev, cache, kind, kv_heads, d, page):
    """Enough tokens of few heads that waves take several: neighbours of one sequence
    and of others, empty ones between, tokens before position 0, pages outside the
    cache, rows of no sequence in front of the first and behind the last."""
    g = torch.Generator().manual_seed(page)
    i = lambda a, b, *n: torch.randint(a, b, n, generator=g, dtype=torch.int32)  # noqa: E731
    seqs, num_pages, width = 3000, 50, 9
    q = i(0, 12, seqs) * (i(0, 4, seqs) > 0)
    q[100], q[101:400] = 200, 0
    kv = torch.clamp(q + i(-2, 2 * page, seqs), min=0, max=width * page)
    table = i(-1, num_pages + 1, seqs, width)
    off = torch.cat([torch.zeros(1, dtype=torch.int32), q.cumsum(0).int()]) + 3
    tokens = int(off[-1]) + 6
    assert tokens > 8192
    if cache == "u8":
        kp, vp = (i(0, 256, num_pages, page, kv_heads, d).to(torch.uint8) for _ in "kv")
        ks, vs = (i(0, 256, num_pages, kv_heads, page).to(torch.uint8) for _ in "kv")
        whole = [Q.values(p, s.transpose(1, 2)) for p, s in ((kp, ks), (vp, vs))]
        extra = {"k_scales": ks.to(torch_dev), "v_scales": vs.to(torch_dev)}
    else:
        kp, vp = (torch.randn(num_pages, page, kv_heads, d, generator=g).to(P.TYPES[cache]) for _ in "kv")
        whole, extra = [kp.float(), vp.float()], {}
    seq = torch.repeat_interleave(torch.arange(seqs), q.long())
    pos = kv[seq] - (off[seq + 1] - torch.arange(3, tokens - 6))
    there = pos >= 0
    at = table[seq, pos.clamp(min=0) // page].long()
    good = there & (at >= 0) & (at < num_pages)
    status = torch.zeros(1, dtype=torch.int32, device=torch_dev)
    out = [torch.full((tokens, kv_heads, d), 7.0, dtype=P.TYPES[kind], device=torch_dev) for _ in "kv"]
    _gh().paged_read(kp.to(torch_dev), vp.to(torch_dev), table.to(torch_dev), off.to(torch_dev), kv.to(torch_dev),
                     k_out=out[0], v_out=out[1], status=status, **extra)
    for got, values in zip(out, whole):
        want = torch.full((tokens, kv_heads, d), 7.0)
        rows = torch.where(good[:, None, None], values[at.clamp(0, num_pages - 1), pos.clamp(min=0) % page], 0.0)
        want[3:-6] = torch.where(there[:, None, None], rows, 7.0)
        assert torch.equal(got.cpu(), want.to(P.TYPES[kind]))
    assert int(status) == (0 if there.all() else 1) + (0 if (good | ~there).all() else 2) == 3


@pytest.mark.parametrize("layout,steps_like", [("heads", "rows"), ("rows", "pages"), ("heads", "pages")])
def test_layouts(torch_dev, layout, steps_like):
    b = Q.batch([5, 1], [21, 9], kind="f16", heads=4, kv_heads=2, d=64, page=8, seed=3, layout=layout, steps_like=steps_like)
    _, x = _append(b, torch_dev)
    after = {**b, **_expected(b)}
    for n in ("k_pages", "v_pages", "k_scales", "v_scales"):
        assert torch.equal(x[n].cpu(), after[n]), n
    _check(after, torch_dev, x=x)


# ---- attention ----------------------------------------------------------------------

def _check(b, dev, *, x=None, scale=None, causal=True, window=0, max_kv=None, **kw):
    """The bound of _paged.attention covers this form too: q has its bits to 2^-23 (two
    pieces; 16-bit q all of them), P as two pieces to 2^-23, and as one to 2^-11, which
    is at most half a step of a 16-bit type.  Results of f16 below 2^-14 lie 2^-24
    apart: their rounding is off by up to 2^-25 whatever their size."""
    want, bound = P.attention(Q.plain(b), scale=scale, causal=causal, window=window)
    bound = bound + (2.0 ** -25 if b["q"].dtype == torch.float16 else 0.0)
    x = Q.to(b, dev) if x is None else x
    out = torch.full_like(x["q"], 3.0)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    _gh().paged_attention(x["q"], *P.args(x), scale=scale, causal=causal, window=window, max_kv_len=max_kv, out=out,
                          status=status, **Q.scales(x), **kw)
    got = out.cpu().double()
    live = ~want.isnan()
    assert ((got - want).abs() <= bound)[live].all(), float(((got - want).abs() / bound)[live].max())
    assert (got[~live] == 3.0).all() and int(status) == 0
    return out


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("heads,kv_heads,d", [(4, 4, 64), (8, 2, 128), (5, 1, 80), (7, 1, 32), (6, 2, 96), (16, 1, 16),
                                              (3, 3, 48), (20, 1, 112)])
@pytest.mark.parametrize("page", [16, 5])
def test_single_tokens(torch_dev, kind, heads, kv_heads, d, page):
    kv = [1, 2, 31, 33, 300, 65, 127, 1030]
    b = Q.batch([1] * len(kv), kv, kind=kind, heads=heads, kv_heads=kv_heads, d=d, page=page, pad=1, seed=d + page)
    _check(b, torch_dev)
    _check(b, torch_dev, window=40, scale=-0.3)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("heads,kv_heads,d", [(32, 8, 128), (28, 4, 128), (48, 2, 64), (20, 5, 80)])
def test_single_tokens_alone(torch_dev, kind, heads, kv_heads, d):
    """Many rows, one token to a sequence: tiles of 16 rows whatever their number,
    groups that cross them, more rows than a tile."""
    kv = [1, 40, 700, 2100, 129, 64]
    b = Q.batch([1] * len(kv), kv, kind=kind, heads=heads, kv_heads=kv_heads, d=d, page=24, seed=d + heads)
    _check(b, torch_dev)
    _check(b, torch_dev, window=100, max_kv=2100)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("heads,kv_heads,d", [(4, 4, 64), (8, 2, 128), (5, 1, 80), (6, 2, 96), (4, 1, 16)])
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 70), (False, 0), (False, 100)])
def test_chunks(torch_dev, kind, heads, kv_heads, d, causal, window):
    q, kv = [150, 1, 70, 0, 200, 33], [150, 90, 333, 7, 260, 33]
    for page in (32, 12):
        b = Q.batch(q, kv, kind=kind, heads=heads, kv_heads=kv_heads, d=d, page=page, seed=d + page)
        _check(b, torch_dev, causal=causal, window=window)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("heads,kv_heads,d", [(4, 4, 64), (8, 2, 128), (5, 1, 80), (6, 2, 96), (4, 1, 16), (7, 1, 32)])
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 300)])
def test_chunks_over_many_keys(torch_dev, kind, heads, kv_heads, d, causal, window):
    """Enough rows and keys for tiles of many rows whatever the heads, beside single
    tokens and an empty sequence."""
    b = Q.batch([701, 1, 0, 303, 2], [2500, 900, 0, 310, 2], kind=kind, heads=heads, kv_heads=kv_heads, d=d, page=16)
    _check(b, torch_dev, causal=causal, window=window)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("q,kv", [([1], [9000]), ([3, 1], [5000, 40]), ([600], [3000]), ([300, 1, 1], [2500, 2600, 8])])
def test_long_axes_in_parts(torch_dev, kind, q, kv):
    b = Q.batch(q, kv, kind=kind, heads=4, kv_heads=1, d=64, page=16, seed=5)
    a = _check(b, torch_dev)
    assert torch.equal(a, _check(b, torch_dev))  # and again the same
    _check(b, torch_dev, max_kv=max(kv))
    _check(b, torch_dev, max_kv=64)  # a wrong length: split otherwise
    gh = _gh()
    x = Q.to(b, torch_dev)
    n = gh.paged_attention_workspace_size(x["q"], *P.args(x))
    ws = torch.full((max(n, 16),), 255, dtype=torch.uint8, device=torch_dev)
    assert torch.equal(_check(b, torch_dev, workspace=ws), a)


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("heads,kv_heads,d,window", [(32, 8, 128, 0), (64, 64, 48, 5000), (48, 6, 80, 0)])
def test_long_prompts(torch_dev, kind, heads, kv_heads, d, window):
    """Enough rows and keys for the largest tiles, ragged, in parts, with a single token beside
    them; the reference and the bound of _paged.attention head by head on the GPU."""
    q_lens, kv_lens = [2070, 1, 77], [5200, 4500, 4200]
    b = Q.batch(q_lens, kv_lens, kind=kind, heads=heads, kv_heads=kv_heads, d=d, page=32, seed=d)
    x = Q.to(b, torch_dev)
    got = _gh().paged_attention(x["q"], *P.args(x), window=window, **Q.scales(x))
    flat = Q.plain(b)
    u, h = 2.0 ** -24, P.half_step(b["q"].dtype)
    at = 0
    for s, (n, kv) in enumerate(zip(q_lens, kv_lens)):
        k, v = (t.to(torch_dev) for t in P.rows_of(flat, s))
        pos = torch.arange(kv - n, kv, device=torch_dev)[:, None]
        j = torch.arange(kv, device=torch_dev)[None]
        hidden = (j > pos) | ((j <= pos - window) if window else False)
        for i in range(0, heads, 5):
            q = x["q"][at:at + n, i].double()
            kk, vv = k[:, i * kv_heads // heads].t().contiguous(), v[:, i * kv_heads // heads].contiguous()
            p = torch.softmax((q @ kk / math.sqrt(d)).masked_fill(hidden, -math.inf), -1)
            want, size = p @ vv, p @ vv.abs()
            delta = u * (d + 8) / math.sqrt(d) * (q.abs() @ kk.abs()).masked_fill(hidden, 0).amax(-1, keepdim=True)
            bound = h * want.abs() + size * (h + 2 * delta + 2.0 ** -21 + kv * u)
            assert ((got[at:at + n, i].double() - want).abs() <= bound).all(), (s, i)
        at += n


def test_pages_of_one_row(torch_dev):
    """More pages than a workgroup looks up at once."""
    for kv, q in ((1500, 1), (2300, 40)):
        b = Q.batch([q], [kv], kind="bf16", heads=4, kv_heads=1, d=32, page=1, seed=6)
        _check(b, torch_dev)


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("size", [2.0 ** -14, 2.0 ** -20, 300.0, 3e3])
def test_rows_of_any_size(torch_dev, kind, size):
    """Steps at the ends of their range; values whose f16 is subnormal.  (The bound goes
    with |q||k| and |V|.)"""
    b = Q.batch([1, 140], [200, 300], kind=kind, heads=2, kv_heads=1, d=64, page=16, seed=8, size=size)
    _check(b, torch_dev, scale=0.125 / size)


@pytest.mark.parametrize("kind,size", [("f32", 1e-30), ("f32", 1e25), ("bf16", 1e-30), ("bf16", 1e25), ("f16", 3e-6),
                                       ("f16", 1e4)])
def test_queries_of_any_size(torch_dev, kind, size):
    """Tiny f16 queries are subnormal as they come, with the bits that they have."""
    b = Q.batch([1, 140], [200, 300], kind=kind, heads=2, kv_heads=1, d=64, page=16, seed=9)
    b["q"] = (b["q"].float() * size).to(b["q"].dtype)
    _check(b, torch_dev, scale=0.125 / size)


@pytest.mark.parametrize("q_len", [1, 150])
def test_queries_that_are_not_finite(torch_dev, q_len):
    """Such a row is NaN; the others are not touched by it."""
    b = Q.batch([q_len, 1], [200, 50], kind="bf16", heads=4, kv_heads=2, d=64, page=16, seed=10)
    want, bound = P.attention(Q.plain(b))
    for bad in (float("nan"), float("inf"), -float("inf")):
        x = Q.to(b, torch_dev)
        x["q"][0, 1, 5] = bad
        got = _gh().paged_attention(x["q"], *P.args(x), **Q.scales(x)).cpu().double()
        assert got[0, 1].isnan().all()
        got[0, 1] = want[0, 1]
        assert ((got - want).abs() <= bound).all()


def test_bad_pages_and_lengths(torch_dev):
    """A page outside the cache reads as zeros, a length beyond the table is cut;
    both are reported."""
    gh = _gh()
    for q_len, page in ((1, 16), (1, 6), (130, 16)):
        b = Q.batch([q_len], [160], kind="f32", heads=2, kv_heads=1, d=32, page=page, seed=11)
        flat = Q.plain(b)
        for bad in (-1, 10 ** 7):
            x = Q.to(b, torch_dev)
            x["page_table"][0, 1] = bad
            zero = {**flat, "k_pages": flat["k_pages"].clone(), "v_pages": flat["v_pages"].clone()}
            for n in ("k_pages", "v_pages"):
                zero[n][int(b["page_table"][0, 1])] = 0
            want, bound = P.attention(zero)
            status = torch.zeros(1, dtype=torch.int32, device=torch_dev)
            got = gh.paged_attention(x["q"], *P.args(x), status=status, **Q.scales(x)).cpu().double()
            assert int(status) == 2 and ((got - want).abs() <= bound).all()
        x = Q.to(b, torch_dev)
        x["kv_lens"][0] = 10 ** 6
        status.zero_()
        gh.paged_attention(x["q"], *P.args(x), status=status, **Q.scales(x))
        assert int(status) & 1
    # pages before a window may be gone
    b = Q.batch([1], [160], kind="bf16", heads=2, kv_heads=1, d=32, page=16, seed=12)
    gone = {**b, "page_table": b["page_table"].clone()}
    gone["page_table"][0, :7] = -1
    want, bound = P.attention(Q.plain(b), window=32)
    x = Q.to(gone, torch_dev)
    status.zero_()
    got = gh.paged_attention(x["q"], *P.args(x), window=32, status=status, **Q.scales(x)).cpu().double()
    assert int(status) == 0 and ((got - want).abs() <= bound).all()


def test_many_sequences(torch_dev):
    """More than a wave's round of the search, empty ones among them."""
    g = torch.Generator().manual_seed(13)
    kv = torch.randint(1, 90, (150,), generator=g).tolist()
    q = [min(n, int(x)) for n, x in zip(kv, torch.randint(0, 4, (150,), generator=g))]
    b = Q.batch(q, kv, kind="f16", heads=4, kv_heads=2, d=64, page=16, pad=3, seed=13)
    _check(b, torch_dev)
    _append_and_check = _expected(b)
    _, x = _append(b, torch_dev)
    for n, t in _append_and_check.items():
        assert torch.equal(x[n].cpu(), t), n


def test_nothing_to_do(torch_dev):
    gh = _gh()
    b = Q.batch([0, 0], [0, 4], kind="bf16", heads=2, kv_heads=2, d=32, page=4, seed=14)
    x = Q.to(b, torch_dev)
    assert gh.paged_attention(x["q"], *P.args(x), **Q.scales(x)).shape == (0, 2, 32)
    gh.paged_append(*P.args(x), x["k"], x["v"], q=x["q"], **Q.scales(x))
    assert gh.paged_read(*P.args(x), **Q.scales(x))[0].shape == (0, 2, 32)


def test_out_on_q(torch_dev):
    b = Q.batch([1, 140], [200, 300], kind="bf16", heads=4, kv_heads=2, d=64, page=16, seed=15)
    x = Q.to(b, torch_dev)
    want = _gh().paged_attention(x["q"], *P.args(x), **Q.scales(x))
    _gh().paged_attention(x["q"], *P.args(x), out=x["q"], **Q.scales(x))
    assert torch.equal(x["q"], want)


# ---- steps ---------------------------------------------------------------------------

@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_steps_of_a_layer(torch_dev, kind):
    """step_paged over an 8-bit cache with norms, prompt and single tokens, against the
    same formulas on the same projections: the cached rows are the rule's on the layer's
    own projections, and the attention is that of the rows that the cache returns."""
    gh = _gh()
    torch.manual_seed(16)
    e, heads, dt = 128, 4, P.TYPES[kind]
    m = gh.MultiHeadAttention(e, heads)
    m.eval()
    m.quantize_grouped(32)
    m.enable_qk_norm(1e-5)
    m.q_norm += 0.2 * torch.randn_like(m.q_norm)
    m.k_norm += 0.2 * torch.randn_like(m.k_norm)
    assert len(m.parameters()) == 10
    cos, sin = (t.to(torch_dev) for t in P.angles(64, e // heads))
    c = gh.PagedKVCache(20, 8, heads, e // heads, dtype=torch.uint8)
    ids = [c.add(), c.add()]
    past = {i: torch.empty(0, e, dtype=dt) for i in ids}
    for counts in ([30, 5], [1, 1], [2, 20], [1, 1]):
        new = [(torch.randn(n, e) * 0.4).to(dt) for n in counts]
        x = torch.cat(new).to(torch_dev)
        got = m.step_paged(x, c, c.extend(ids, counts), cos=cos, sin=sin)
        q, k, v = (m.w4[i](x).view(-1, heads, e // heads).cpu() for i in range(3))
        y, bounds, at = [], [], 0
        for i, n in zip(ids, counts):
            first = len(past[i])
            past[i] = torch.cat((past[i], x[at:at + n].cpu()))
            kk, vv = (t.cpu() for t in c.read(i))
            assert kk.shape == (first + n, heads, e // heads)
            rows = torch.stack([Q.turned(Q.normed(k[at + j], m.k_norm.cpu(), 1e-5), first + j, cos.cpu(), sin.cpu(), False)
                                for j in range(n)])
            assert torch.equal(kk[first:], Q.values(*Q.quantise(rows)))
            assert torch.equal(vv[first:], Q.values(*Q.quantise(v[at:at + n])))
            qq = torch.stack([Q.turned(Q.normed(q[at + j], m.q_norm.cpu(), 1e-5), first + j, cos.cpu(), sin.cpu(), False)
                              for j in range(n)]).to(dt)
            one = {"q": qq, "q_offsets": torch.tensor([0, n]), "kv_lens": torch.tensor([first + n]), "page": first + n,
                   "page_table": torch.zeros(1, 1, dtype=torch.int32), "k_pages": kk[None], "v_pages": vv[None]}
            o, bound = P.attention(one)
            y.append(o.flatten(1))
            bounds.append(bound.flatten(1))
            at += n
        w, bias = m.w4[3].dequantize().double().cpu(), m.w4[3].bias.double().cpu()
        y, bounds = torch.cat(y), torch.cat(bounds)
        want = y @ w.t() + bias
        # attention's own bound through the projection, whose sums of 128 terms are in
        # fp32 and which rounds once
        room = (bounds + 2 * P.half_step(dt) * y.abs() + 136 * 2.0 ** -24 * y.abs()) @ w.abs().t()
        assert ((got.cpu().double() - want).abs() <= room + P.half_step(dt) * want.abs() + 2.0 ** -22).all()
    for call in (lambda: m.step(torch.zeros(1, 1, e, device=torch_dev), gh.KVCache(1, 4, e)),
                 lambda: m.forward(torch.zeros(1, 1, e, device=torch_dev))):
        with pytest.raises(gh.GhostFlowError, match="step_paged"):
            call()


def test_a_captured_step(torch_dev):
    """Append, read and attention in one graph, replayed after lengths, tables and
    values changed, with eager work between: every replay is the eager result."""
    gh = _gh()
    b = Q.batch([1, 1, 1], [700, 20, 333], kind="bf16", heads=8, kv_heads=2, d=64, page=16, seed=17, spare=8)
    x = Q.to(b, torch_dev)
    w = (1 + 0.1 * torch.randn(64)).to(torch_dev)
    out, back = torch.zeros_like(x["q"]), [torch.zeros_like(x["k"]) for _ in range(2)]
    size = gh.paged_attention_workspace_size(x["q"], *P.args(x))
    ws = torch.empty(max(size, 16), dtype=torch.uint8, device=torch_dev)
    q_out = torch.zeros_like(x["q"])

    def step():
        gh.paged_append(*P.args(x), x["k"], x["v"], q=x["q"], q_out=q_out, q_norm=w, k_norm=w, **Q.scales(x))
        gh.paged_attention(q_out, *P.args(x), out=out, workspace=ws, **Q.scales(x))
        gh.paged_read(*P.args(x), k_out=back[0], v_out=back[1], **Q.scales(x))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        step()
    for n in range(4):
        x["k"].copy_(torch.randn(x["k"].shape))
        x["q"].copy_(torch.randn(x["q"].shape))
        x["kv_lens"].copy_(torch.tensor([700 - 90 * n, 20 + n, 333], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (out, *back, q_out, x["k_pages"], x["k_scales"])]
        for t in (out, *back, q_out):
            t.zero_()
        step()
        torch.cuda.synchronize()
        for a, t in zip(got, (out, *back, q_out, x["k_pages"], x["k_scales"])):
            assert torch.equal(a, t)


def test_two_streams_at_once(torch_dev):
    """Calls without a workspace on two streams, each over its own cache."""
    gh = _gh()
    work = []
    for seed in (18, 19):
        b = Q.batch([1, 1], [3000, 900], kind="bf16", heads=8, kv_heads=2, d=128, page=16, seed=seed)
        x = Q.to(b, torch_dev)
        work.append((x, gh.paged_attention(x["q"], *P.args(x), **Q.scales(x)), torch.cuda.Stream()))
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(5):
        for i, (x, _, s) in enumerate(work):
            with torch.cuda.stream(s):
                outs[i].append(gh.paged_attention(x["q"], *P.args(x), **Q.scales(x)))
    torch.cuda.synchronize()
    for i, (_, want, _) in enumerate(work):
        assert all(torch.equal(o, want) for o in outs[i])


def test_offsets_beyond_32_bits(torch_dev):
    """Pages whose bytes lie beyond 2^32 from the cache's first."""
    gh = _gh()
    pages, page, hkv, d = 70000, 64, 8, 128  # 4.6 GB each
    k = torch.empty(pages, page, hkv, d, dtype=torch.uint8, device=torch_dev)
    v = torch.empty_like(k)
    ks = torch.empty(pages, hkv, page, dtype=torch.uint8, device=torch_dev)
    vs = torch.empty_like(ks)
    table = torch.tensor([[pages - 1, 3, pages - 2]], dtype=torch.int32, device=torch_dev)
    g = torch.Generator(device=torch_dev).manual_seed(20)
    new = [torch.randn(150, hkv, d, generator=g, device=torch_dev) for _ in range(2)]
    off, lens = (torch.tensor(t, dtype=torch.int32, device=torch_dev) for t in ([0, 150], [150]))
    gh.paged_append(k, v, table, off, lens, *new, k_scales=ks, v_scales=vs)
    got = gh.paged_read(k, v, table, off, lens, tokens=150, k_scales=ks, v_scales=vs)
    want = [Q.values(*Q.quantise(t.cpu())) for t in new]
    assert all(torch.equal(a.cpu(), b) for a, b in zip(got, want))
    for n in (1, 150):
        q = torch.randn(n, hkv, d, generator=g, device=torch_dev)
        o = gh.paged_attention(q, k, v, table, off.new_tensor([0, n]), lens, k_scales=ks, v_scales=vs).cpu().double()
        score = torch.einsum("qhd,khd->hqk", q.cpu().double(), want[0].double()) / math.sqrt(d)
        hidden = torch.arange(150)[None] > torch.arange(150 - n, 150)[:, None]
        p = torch.softmax(score.masked_fill(hidden, -math.inf), -1)
        ref = torch.einsum("hqk,khd->qhd", p, want[1].double())
        # scores: sums of 128 terms of at most some 4 x 4 in fp32, over sqrt(128)
        assert (o - ref).abs().max() <= 2 * 136 * 2.0 ** -24 * 16 * 128 / math.sqrt(d)


# ---- what has one answer whatever the sizes ---------------------------------------------

@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("heads,kv_heads,d,q,kv", [(8, 2, 128, 600, 2500), (8, 4, 64, 700, 2600), (32, 8, 128, 2048, 4200)])
def test_prompts_round_as_their_type_does(torch_dev, kind, heads, kv_heads, d, q, kv):
    """The mean square error against 64 bits is that of the output's own rounding.  What a
    rounding of the weights to f16 adds: a value with mantissa m is off by 2^-10 / sqrt(12) / m
    (root of the mean square), a bf16 output by 2^-7 / sqrt(12) / m, so at most (2.8e-4 / 1.1e-3)^2
    / 2 = 3.2% where every weight has the smallest mantissa and every output the largest, and
    0.8% for mantissas alike; for an f16 output it would be 41%."""
    b = Q.batch([q], [kv], kind=kind, heads=heads, kv_heads=kv_heads, d=d, page=32, seed=d + q)
    x = Q.to(b, torch_dev)
    got = _gh().paged_attention(x["q"], *P.args(x), **Q.scales(x)).double()
    k, v = (t.to(torch_dev) for t in P.rows_of(Q.plain(b), 0))
    hidden = torch.arange(kv, device=torch_dev)[None] > torch.arange(kv - q, kv, device=torch_dev)[:, None]
    for i in range(0, heads, 3):
        kk, vv = k[:, i * kv_heads // heads].t().contiguous(), v[:, i * kv_heads // heads].contiguous()
        p = torch.softmax((x["q"][:, i].double() @ kk / math.sqrt(d)).masked_fill(hidden, -math.inf), -1)
        want = p @ vv
        own = (want.to(P.TYPES[kind]).double() - want).norm()
        assert (got[:, i] - want).norm() <= 1.04 * own, (i, float((got[:, i] - want).norm() / own))


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("scale", [0.0, 1e-30, -1e-38])
@pytest.mark.parametrize("size", [1.0, 1e-4, 1e-6, 1e-30, 1e30, 1e37])
def test_scales_of_next_to_nothing(torch_dev, kind, scale, size):
    """Every row is the mean of the values that it sees, whatever its queries' size: equal
    weights, which lose nothing in any type; their sum in fp32, one rounding."""
    if kind == "f16" and size > 1e4 or scale and size > 1:
        return
    for q, kv, page in (([1, 1], [200, 33], 16), ([1, 140], [200, 301], 12), ([400], [1501], 16)):
        b = Q.batch(q, kv, kind=kind, heads=8, kv_heads=4, d=64, page=page, seed=21)
        b["q"] = (b["q"].float() * size).to(b["q"].dtype)
        x, flat = Q.to(b, torch_dev), Q.plain(b)
        for window in (0, 70):
            got = _gh().paged_attention(x["q"], *P.args(x), scale=scale, window=window, **Q.scales(x)).cpu().double()
            at = 0
            for s, (m, n) in enumerate(zip(q, kv)):
                v = P.rows_of(flat, s)[1].repeat_interleave(2, 1)
                hi = torch.arange(n - m + 1, n + 1)
                lo = (hi - window).clamp(min=0) if window else 0 * hi
                sums = [torch.cat((0 * t[:1], t)).cumsum(0) for t in (v, v.abs())]
                want, mean = ((t[hi] - t[lo]) / (hi - lo)[:, None, None] for t in sums)
                bound = P.half_step(b["q"].dtype) * want.abs() + mean * (2.0 ** -21 + n * 2.0 ** -24) + 2.0 ** -25
                assert ((got[at:at + m] - want).abs() <= bound).all(), (s, window)
                at += m


def _many(seqs, longest, heads, kv_heads, d, page, kind, dev, seed):
    """One new token each of ragged sequences whose pages lie anywhere, the cache any codes
    and steps of usual values, made on the device."""
    g = torch.Generator(device=dev).manual_seed(seed)
    i = lambda lo, hi, *n: torch.randint(lo, hi, n, generator=g, device=dev)  # noqa: E731
    lens = i(longest // 4, longest + 1, seqs)
    lens[0], lens[1] = longest, 1
    pages = (lens + page - 1) // page
    total, width = int(pages.sum()), int(pages.max())
    order = torch.randperm(total, generator=g, device=dev).int()
    col = torch.arange(width, device=dev)
    table = torch.full((seqs, width), -1, dtype=torch.int32, device=dev)
    used = col < pages[:, None]
    table[used] = order[((pages.cumsum(0) - pages)[:, None] + col)[used]]
    x = {"page_table": table, "kv_lens": lens.int(), "q_offsets": torch.arange(seqs + 1, device=dev).int()}
    for n in "kv":
        x[n + "_pages"] = i(0, 256, total, page, kv_heads, d).to(torch.uint8)
        x[n + "_scales"] = i(96, 104, total, kv_heads, page).to(torch.uint8)
    x["q"] = torch.randn(seqs, heads, d, generator=g, device=dev).to(P.TYPES[kind])
    return x


@pytest.mark.parametrize("kind", ["bf16", "f32"])
@pytest.mark.parametrize("page", [16, 20])
@pytest.mark.parametrize("seqs,longest,heads,kv_heads,d,window", [
    (64, 4096, 32, 8, 128, 0), (64, 4096, 32, 8, 128, 2500), (70, 4300, 16, 8, 64, 0), (100, 2600, 12, 6, 80, 0),
    (310, 2300, 8, 2, 64, 0), (150, 3000, 16, 4, 96, 2200)])
def test_heads_side_by_side(torch_dev, kind, page, seqs, longest, heads, kv_heads, d, window):
    """Single tokens of so many long sequences that four, or two, key/value heads share a
    workgroup: three workgroups to a CU leave each 1024 keys of a head and more.  Every head
    of every sequence against 64 bits, with the bound of _paged.attention."""
    x = _many(seqs, longest, heads, kv_heads, d, page, kind, torch_dev, seqs + page)
    status = torch.zeros(1, dtype=torch.int32, device=torch_dev)
    got = _gh().paged_attention(x["q"], *P.args(x), window=window, max_kv_len=longest, status=status, **Q.scales(x))
    steps = Q.STEPS.double().to(torch_dev)
    u, h = 2.0 ** -24, P.half_step(x["q"].dtype)
    for s in range(seqs):
        n = int(x["kv_lens"][s])
        lo = max(0, n - window) if window else 0
        at = x["page_table"][s, :-(-n // page)].long()
        k, v = (((x[c + "_pages"][at].double() - 128) * steps[x[c + "_scales"][at].transpose(1, 2).long()][..., None])
                .flatten(0, 1)[lo:n].transpose(0, 1).contiguous() for c in "kv")  # [kv_heads, keys, d]
        q = x["q"][s].double().view(kv_heads, -1, d)
        kt = k.transpose(1, 2).contiguous()
        p = torch.softmax(q @ kt / math.sqrt(d), -1)
        want, size = p @ v, p @ v.abs()
        delta = u * (d + 8) / math.sqrt(d) * (q.abs() @ kt.abs()).amax(-1, keepdim=True)
        bound = h * want.abs() + size * (h + 2 * delta + 2.0 ** -21 + (n - lo) * u)
        assert ((got[s].double().view(kv_heads, -1, d) - want).abs() <= bound).all(), s
    assert int(status) == 0


def test_every_border_between_steps(torch_dev):
    """Rows whose largest magnitude is 127 of each of the 208 steps, and its neighbours in fp32."""
    g = torch.Generator().manual_seed(22)
    most = 127.0 * Q.STEPS
    most = torch.stack((most, torch.nextafter(most, torch.tensor(0.0)), torch.nextafter(most, torch.tensor(1e6))), 1).flatten()[:-1]
    n, d = len(most), 32  # (but the largest's upper neighbour, which no step holds)
    rows = (torch.rand(n, 2, d, generator=g) * 2 - 1) * most[:, None, None]
    rows[torch.arange(n), :, torch.arange(n) % d] = torch.stack((most, -most), 1)
    b = Q.batch([n], [n], kind="f32", heads=2, kv_heads=2, d=d, page=16, seed=22)
    b["k"], b["v"] = rows, rows.flip(0)
    status = torch.zeros(1, dtype=torch.int32, device=torch_dev)
    _, x = _append(b, torch_dev, status=status)
    for name, t in _expected(b).items():
        assert torch.equal(x[name].cpu(), t), name
    assert int(status) == 0


@pytest.mark.parametrize("name", ["page_table", "q_offsets", "kv_lens"])
def test_the_wrong_argument_is_named(torch_dev, name):
    gh = _gh()
    b = Q.to(Q.batch([1, 1], [20, 9], kind="bf16", heads=2, kv_heads=1, d=32, page=16, seed=23), torch_dev)
    twice = torch.stack((b[name], b[name]), -1)
    for bad in (b[name].long(), b[name].cpu(), twice[..., 0]):
        x = {**b, name: bad}
        for call in (lambda: gh.paged_attention(x["q"], *P.args(x), **Q.scales(x)),
                     lambda: gh.paged_append(*P.args(x), x["k"], x["v"], **Q.scales(x)),
                     lambda: gh.paged_read(*P.args(x), tokens=2, **Q.scales(x))):
            with pytest.raises(gh.GhostFlowError, match=rf"(?<!and ){name} must be a contiguous int32 tensor"):
                call()


def test_a_layer_says_what_it_could_not_write(torch_dev):
    """step_paged's status: values past the largest code's, and NaN, set bit 2; a page outside
    the cache bit 1."""
    gh = _gh()
    torch.manual_seed(24)
    m = gh.MultiHeadAttention(64, 2)
    m.eval()
    status = torch.zeros(1, dtype=torch.int32, device=torch_dev)
    for scale, bits in ((1.0, 0), (1e7, 4), (float("nan"), 4)):
        c = gh.PagedKVCache(4, 8, 2, 32, dtype=torch.uint8)
        x = torch.randn(3, 64, device=torch_dev) * scale
        status.zero_()
        m.step_paged(x, c, c.extend([c.add()], [3]), status=status)
        assert int(status) == bits, scale
    c = gh.PagedKVCache(4, 8, 2, 32)
    batch = c.extend([c.add()], [3])
    batch.page_table.fill_(9)
    status.zero_()
    m.step_paged(torch.randn(3, 64, device=torch_dev), c, batch, status=status)
    assert int(status) == 2
