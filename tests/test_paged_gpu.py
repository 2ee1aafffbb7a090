"""Paged append (with rotary positions) and paged attention on the GPU against
the plain form in 64 bits (_paged.py): types, head layouts, page sizes and
layouts, ragged and empty sequences, windows, masked rows.  Rows of the pages
that hold no position are NaN, so any use of them shows."""
import math

import pytest
import torch

import _paged as P

pytestmark = pytest.mark.gpu


def _gh():
    import ghostflow_hip
    return ghostflow_hip


def _check(got, want, bound):
    got = got.double().cpu()
    live = ~torch.isnan(want)
    err = (got - want).abs()
    assert torch.isfinite(got[live]).all()
    bad = live & (err > bound)
    assert not bad.any(), (int(bad.sum()), float(err[bad].max()), float(bound[bad].min()))


def _attend(dev, b, **kw):
    gh = _gh()
    x = P.to(b, dev)
    out = torch.full_like(x["q"], 7.0)
    hint = kw.pop("max_kv_len", None)
    got = gh.paged_attention(x["q"], *P.args(x), out=out, max_kv_len=hint, **kw)
    torch.cuda.synchronize()
    return got


# lengths: one token; decode; chunks that end inside pages and tiles; no past;
# sequences without new tokens or without any position; more tokens than keys
LENS = [
    ([1], [1]),
    ([1], [517]),
    ([1, 1, 1, 1, 1], [33, 1, 700, 64, 129]),
    ([5, 0, 1, 3], [5, 40, 65, 300]),
    ([70, 1, 33], [70, 260, 100]),
    ([200], [1000]),
    ([300, 1, 2, 0, 130], [900, 700, 40, 5, 130]),
    ([140, 1, 2, 1, 0, 1], [200, 500, 300, 700, 4, 1000]),
    ([0, 0, 2, 0], [10, 0, 9, 0]),
    ([4, 9], [2, 0]),
]
HEADS = [(4, 4, 64), (8, 2, 128), (6, 1, 80), (3, 3, 8), (40, 2, 32), (7, 1, 128), (2, 2, 96), (40, 1, 64)]


@pytest.mark.parametrize("types", P.PAIRS, ids="/".join)
@pytest.mark.parametrize("lens", LENS, ids=lambda v: "-".join(map(str, v[0])))
def test_attention_lengths(torch_dev, types, lens):
    for heads, kv_heads, d in ((8, 2, 128), (4, 4, 64)):
        b = P.batch(*lens, heads=heads, kv_heads=kv_heads, d=d, page=16, types=types, seed=1)
        _check(_attend(torch_dev, b), *P.attention(b))


@pytest.mark.parametrize("types", P.PAIRS, ids="/".join)
@pytest.mark.parametrize("heads", HEADS, ids=lambda v: "-".join(map(str, v)))
def test_attention_heads(torch_dev, types, heads):
    h, hkv, d = heads
    b = P.batch([1, 40, 3], [300, 90, 77], heads=h, kv_heads=hkv, d=d, page=16, types=types, seed=2)
    _check(_attend(torch_dev, b), *P.attention(b))


# prompts of many heads, which fill the GPU with the tiles of fp32 prompts too
MANY = dict(heads=32, kv_heads=32, page=24, pad=2)


@pytest.mark.parametrize("types", P.PAIRS, ids="/".join)
@pytest.mark.parametrize("d,causal,window", [(8, True, 90), (64, True, 0), (104, False, 0), (128, True, 0), (128, True, 90)])
def test_attention_of_prompts_of_many_heads(torch_dev, types, d, causal, window):
    b = P.batch([300, 1, 40, 180, 0], [1100, 50, 300, 180, 9], d=d, types=types, seed=d, **MANY)
    _check(_attend(torch_dev, b, causal=causal, window=window), *P.attention(b, causal=causal, window=window))


@pytest.mark.parametrize("types,value", [(("f32", "f32"), float("nan")), (("f32", "f32"), float("inf")),
                                         (("bf16", "bf16"), float("nan"))])
@pytest.mark.parametrize("which", ["k_pages", "v_pages"])
def test_prompts_of_many_heads_do_not_see_later_tokens(torch_dev, types, value, which):
    b = P.batch([520], [700], d=32, types=types, seed=40, **MANY)
    at = 500  # its token is row 320: the rows before see nothing of it
    b[which][b["page_table"][0, at // 24].long(), at % 24] = value
    got = _attend(torch_dev, b)
    want, bound = P.attention(b)
    _check(got[:320], want[:320], bound[:320])
    assert torch.isnan(got[320:520]).all() if value != value else not torch.isfinite(got[320:520]).all()


@pytest.mark.parametrize("types", P.PAIRS, ids="/".join)
@pytest.mark.parametrize("heads", [(33, 1), (64, 1), (40, 1), (96, 2)], ids=lambda v: "-".join(map(str, v)))
def test_one_token_of_more_heads_than_a_few_rows(torch_dev, types, heads):
    for n in (1, 70, 900):
        b = P.batch([1], [n], heads=heads[0], kv_heads=heads[1], d=64, page=16, types=types, seed=n)
        _check(_attend(torch_dev, b), *P.attention(b))


@pytest.mark.parametrize("types", P.PAIRS, ids="/".join)
@pytest.mark.parametrize("page", [1, 3, 16, 48, 64, 1000])
@pytest.mark.parametrize("layout", ["rows", "heads", "pairs"])
def test_attention_pages(torch_dev, types, page, layout):
    b = P.batch([1, 50], [211, 333], heads=4, kv_heads=2, d=64, page=page, types=types, seed=3, layout=layout)
    _check(_attend(torch_dev, b), *P.attention(b))


@pytest.mark.parametrize("types", P.PAIRS, ids="/".join)
@pytest.mark.parametrize("causal,window", [(False, 0), (True, 1), (True, 20), (True, 128), (True, 10 ** 6), (False, 50)])
def test_attention_masks(torch_dev, types, causal, window):
    b = P.batch([1, 90, 2, 4], [400, 300, 2, 3], heads=4, kv_heads=1, d=128, page=16, types=types, seed=4)
    _check(_attend(torch_dev, b, causal=causal, window=window), *P.attention(b, causal=causal, window=window))


@pytest.mark.parametrize("types", P.PAIRS, ids="/".join)
@pytest.mark.parametrize("scale", [0.0, -0.125, 1.0, 1e-30])
def test_attention_scales(torch_dev, types, scale):
    b = P.batch([1, 60], [200, 150], heads=4, kv_heads=2, d=64, page=16, types=types, seed=5)
    _check(_attend(torch_dev, b, scale=scale), *P.attention(b, scale=scale))


@pytest.mark.parametrize("types", P.PAIRS, ids="/".join)
def test_attention_long_axis_is_split_and_any_hint_is_right(torch_dev, types):
    """Few rows over a long axis: the result holds whatever the caller says
    about the longest length, and is the same bits every time."""
    b = P.batch([1, 2, 30], [6001, 257, 3000], heads=4, kv_heads=2, d=128, page=16, types=types, seed=6)
    want = P.attention(b)
    for hint in (None, 6001, 100, 10 ** 9):
        got = _attend(torch_dev, b, max_kv_len=hint)
        _check(got, *want)
        assert torch.equal(got, _attend(torch_dev, b, max_kv_len=hint))


@pytest.mark.parametrize("types", P.PAIRS, ids="/".join)
def test_attention_leaves_padding_and_serves_any_offsets(torch_dev, types):
    """Rows behind the last sequence keep what they held; more sequences than
    a wave has lanes, most without new tokens."""
    b = P.batch([1, 40], [50, 60], heads=4, kv_heads=2, d=64, page=16, types=types, seed=7, pad=9)
    got = _attend(torch_dev, b)
    _check(got[:41], *(x[:41] for x in P.attention(b)))
    assert (got[41:] == 7.0).all()
    lens = [0 if s % 7 else 1 + s % 3 for s in range(300)]
    b = P.batch(lens, [n + s % 50 for s, n in enumerate(lens)], heads=2, kv_heads=2, d=64, page=16, types=types, seed=8)
    _check(_attend(torch_dev, b), *P.attention(b))


@pytest.mark.parametrize("types", P.PAIRS, ids="/".join)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("which", ["k_pages", "v_pages"])
def test_attention_masked_values_do_not_reach_a_row(torch_dev, types, value, which):
    """A value that is not finite in a key that only later tokens see, or only
    earlier ones (window): the others' rows stay as the plain form, which
    leaves that key out, has them."""
    b = P.batch([60, 1], [300, 200], heads=4, kv_heads=2, d=64, page=16, types=types, seed=9)
    page, row = b["page_table"][0, 270 // 16].long(), 270 % 16
    b[which][page, row, 1, 5] = value
    for window in (0, 40):
        want, bound = P.attention(b, window=window)
        got = _attend(torch_dev, b, window=window).double().cpu()
        sees = torch.zeros(61, 4, dtype=torch.bool)
        for t in range(60):
            p = 240 + t
            sees[t, 2:] = p >= 270 and (not window or 270 > p - window)
        fine = ~sees[..., None].expand_as(want)
        assert (got - want).abs()[fine].le(bound[fine]).all()
        # and the rows that see it are finite where the formula's are
        assert torch.equal(torch.isfinite(got[~fine]), torch.isfinite(want[~fine]))


@pytest.mark.parametrize("types", P.PAIRS, ids="/".join)
def test_attention_strided_rows_and_in_place(torch_dev, types):
    """q as a slice of a fused projection, out in a wider tensor; out on q."""
    gh = _gh()
    b = P.batch([1, 40, 5], [300, 90, 77], heads=4, kv_heads=2, d=64, page=16, types=types, seed=10)
    want = P.attention(b)
    x = P.to(b, torch_dev)
    t = x["tokens"]
    fused = torch.zeros(t, 8, 64, dtype=x["q"].dtype, device=torch_dev)
    fused[:, 2:6] = x["q"]
    wide = torch.zeros(t, 6, 64, dtype=x["q"].dtype, device=torch_dev)
    gh.paged_attention(fused[:, 2:6], *P.args(x), out=wide[:, 1:5])
    _check(wide[:, 1:5], *want)
    assert (wide[:, 0] == 0).all() and (wide[:, 5] == 0).all()
    same = x["q"].clone()
    gh.paged_attention(same, *P.args(x), out=same)
    _check(same, *want)


@pytest.mark.parametrize("types", [("bf16", "bf16"), ("f32", "f32")], ids="/".join)
def test_attention_shared_pages(torch_dev, types):
    """Two sequences over one prefix."""
    b = P.batch([3, 20], [200, 250], heads=4, kv_heads=2, d=64, page=16, types=types, seed=11)
    b["page_table"][1, :6] = b["page_table"][0, :6]
    _check(_attend(torch_dev, b), *P.attention(b))


@pytest.mark.parametrize("types", P.PAIRS, ids="/".join)
def test_bad_pages_and_lengths_are_reported(torch_dev, types):
    """A page outside the cache is not touched and sets a bit of status; so
    does a length the table cannot hold.  The other sequences are served."""
    gh = _gh()
    b = P.batch([1, 40, 2], [100, 90, 77], heads=4, kv_heads=2, d=64, page=16, types=types, seed=12)
    want, bound = P.attention(b)
    for bad in (-1, 10 ** 6):
        c = dict(b, page_table=b["page_table"].clone())
        c["page_table"][0, 2] = bad
        x = P.to(c, torch_dev)
        st = torch.zeros(1, dtype=torch.int32, device=torch_dev)
        got = gh.paged_attention(x["q"], *P.args(x), status=st)
        assert int(st) == 2
        _check(got[1:], want[1:], bound[1:])
        st.zero_()
        c["page_table"][0, 6] = bad  # where the new token goes
        x = P.to(c, torch_dev)
        gh.paged_append(*P.args(x), x["k"], x["v"], status=st)
        assert int(st) == 2
    for n in (-5, 10 ** 6):
        c = dict(b, kv_lens=b["kv_lens"].clone())
        c["kv_lens"][0] = n
        x = P.to(c, torch_dev)
        st = torch.zeros(1, dtype=torch.int32, device=torch_dev)
        got = gh.paged_attention(x["q"], *P.args(x), status=st)
        assert int(st) & 1
        _check(got[1:], want[1:], bound[1:])
        st.zero_()
        gh.paged_append(*P.args(x), x["k"], x["v"], status=st)
        assert int(st) == 1


# ---- append --------------------------------------------------------------------------


@pytest.mark.parametrize("types", P.PAIRS, ids="/".join)
@pytest.mark.parametrize("rot,interleaved", [(0, False), (64, False), (64, True), (32, False), (24, True), (8, False)])
@pytest.mark.parametrize("lens", [([1], [1]), ([1, 1, 1], [33, 1, 700]), ([5, 0, 30], [5, 40, 65])],
                         ids=lambda v: "-".join(map(str, v[0])))
def test_append(torch_dev, types, rot, interleaved, lens):
    gh = _gh()
    for heads, kv_heads, d, page, layout in ((4, 2, 64, 16, "rows"), (3, 1, 72, 5, "heads"), (8, 8, 128, 1, "pairs")):
        b = P.batch(*lens, heads=heads, kv_heads=kv_heads, d=d, page=page, types=types, seed=20, pad=3, stale=9.0,
                    layout=layout)
        cos = sin = None
        if rot:
            cos, sin = P.angles(b["page_table"].shape[1] * page, rot)
        x = P.to(b, torch_dev)
        q_out = torch.full_like(x["q"], 5.0)
        dc, ds = (None, None) if cos is None else (cos.to(torch_dev), sin.to(torch_dev))
        r = gh.paged_append(*P.args(x), x["k"], x["v"], q=x["q"], q_out=q_out, cos=dc, sin=ds, interleaved=interleaved)
        assert r is q_out
        got_k, got_v, got_q = x["k_pages"].double().cpu(), x["v_pages"].double().cpu(), q_out.double().cpu()
        want_k, want_v, want_q = b["k_pages"].double(), b["v_pages"].double(), torch.full_like(got_q, 5.0)
        mag_k, mag_q = torch.zeros_like(want_k), torch.zeros_like(want_q)
        for s in range(len(lens[0])):
            a, e, n = int(b["q_offsets"][s]), int(b["q_offsets"][s + 1]), int(b["kv_lens"][s])
            for t in range(a, e):
                p = n - (e - t)
                at = (b["page_table"][s, p // page].long(), p % page)
                want_k[at] = P.turned(b["k"][t], p, cos, sin, interleaved)
                want_v[at] = b["v"][t].double()
                want_q[t] = P.turned(b["q"][t], p, cos, sin, interleaved)
                # two products and a sum in fp32, of at most |a| + |b|
                mag_k[at] = 2 * b["k"][t].abs().double().amax()
                mag_q[t] = 2 * b["q"][t].abs().double().amax()
        hc, ha = P.half_step(x["k_pages"].dtype), P.half_step(x["q"].dtype)
        assert (got_k - want_k).abs().le(hc * want_k.abs() * (1 + 2 ** -10) + 2.0 ** -23 * mag_k).all()
        assert (got_v - want_v).abs().le(hc * want_v.abs()).all()
        assert (got_q - want_q).abs().le(ha * want_q.abs() * (1 + 2 ** -10) + 2.0 ** -23 * mag_q).all()


def test_append_in_place_strided_and_without_q(torch_dev):
    gh = _gh()
    b = P.batch([1, 9], [20, 30], heads=4, kv_heads=2, d=64, page=16, types=("bf16", "bf16"), seed=21, stale=0.0)
    cos, sin = (t.to(torch_dev) for t in P.angles(b["page_table"].shape[1] * 16, 64))
    x = P.to(b, torch_dev)
    q_out = gh.paged_append(*P.args(x), x["k"], x["v"], q=x["q"], cos=cos, sin=sin)
    fused = torch.cat([x["q"], x["k"], x["v"]], 1)
    y = P.to(b, torch_dev)
    q = fused[:, :4]
    assert gh.paged_append(*P.args(y), fused[:, 4:6], fused[:, 6:], q=q, q_out=q, cos=cos, sin=sin) is q
    assert torch.equal(q, q_out) and torch.equal(x["k_pages"], y["k_pages"]) and torch.equal(x["v_pages"], y["v_pages"])
    z = P.to(b, torch_dev)
    assert gh.paged_append(*P.args(z), z["k"], z["v"], cos=cos, sin=sin) is None
    assert torch.equal(x["k_pages"], z["k_pages"]) and torch.equal(x["v_pages"], z["v_pages"])


# ---- together --------------------------------------------------------------------------


@pytest.mark.parametrize("types", P.PAIRS, ids="/".join)
def test_chunks_then_tokens_give_what_one_prompt_gives(torch_dev, types):
    """A prompt in one call, and in chunks followed by single tokens: append
    and attend at every step.  The same keys and probabilities, in other
    tiles: both within the bound of the plain form over the cache."""
    gh = _gh()
    n, page = 150, 16
    b = P.batch([n], [n], heads=8, kv_heads=2, d=64, page=page, types=types, seed=22)
    cos, sin = (t.to(torch_dev) for t in P.angles(b["page_table"].shape[1] * page, 64))
    x = P.to(b, torch_dev)
    q = gh.paged_append(*P.args(x), x["k"], x["v"], q=x["q"], cos=cos, sin=sin)
    out = gh.paged_attention(q, *P.args(x))
    host = dict(b, k_pages=x["k_pages"].cpu(), v_pages=x["v_pages"].cpu(), q=q.cpu())
    want, bound = P.attention(host)
    _check(out, want, bound)
    y = P.to(b, torch_dev)
    at = 0
    for m in [64, 33, 20] + [1] * 33:
        off = torch.tensor([0, m], dtype=torch.int32, device=torch_dev)
        kl = torch.tensor([at + m], dtype=torch.int32, device=torch_dev)
        cache = (y["k_pages"], y["v_pages"], y["page_table"], off, kl)
        r = gh.paged_append(*cache, y["k"][at:at + m], y["v"][at:at + m], q=y["q"][at:at + m], cos=cos, sin=sin)
        assert torch.equal(r, q[at:at + m])
        _check(gh.paged_attention(r, *cache), want[at:at + m], bound[at:at + m])
        at += m
    assert torch.equal(x["k_pages"].nan_to_num(9), y["k_pages"].nan_to_num(9))


def test_captured_step_follows_lengths_and_tables(torch_dev):
    """A decode step captured once and replayed while the sequences grow, a
    second graph with its own workspace beside it, eager work between."""
    gh = _gh()
    types = ("bf16", "bf16")
    b = P.batch([1, 1, 1], [2000, 700, 60], heads=8, kv_heads=2, d=128, page=16, types=types, seed=23, stale=0.0)
    x = P.to(b, torch_dev)
    cos, sin = (t.to(torch_dev) for t in P.angles(b["page_table"].shape[1] * 16, 128))
    streams = [torch.cuda.Stream() for _ in range(2)]
    size = gh.paged_attention_workspace_size(x["q"], *P.args(x))
    assert size > 0
    ws = [torch.empty(size, dtype=torch.uint8, device=torch_dev) for _ in range(2)]
    outs = [torch.empty_like(x["q"]) for _ in range(2)]
    qs = [torch.empty_like(x["q"]) for _ in range(2)]

    def step(i):
        gh.paged_append(*P.args(x), x["k"], x["v"], q=x["q"], q_out=qs[i], cos=cos, sin=sin)
        gh.paged_attention(qs[i], *P.args(x), out=outs[i], workspace=ws[i])

    graphs = []
    for i, s in enumerate(streams):
        s.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            step(i)
        graphs.append(g)
    torch.cuda.synchronize()
    for rep in range(4):
        x["kv_lens"].copy_(torch.tensor([1900 + 7 * rep, 650 + rep, 50 + rep], dtype=torch.int32))
        x["q"].normal_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        want = gh.paged_attention(qs[0], *P.args(x))
        torch.cuda.synchronize()
        assert torch.equal(got[0], want) and torch.equal(got[1], want), rep


@pytest.mark.parametrize("types", P.PAIRS, ids="/".join)
@pytest.mark.parametrize("q_lens", [[1, 1], [40, 1]])
def test_pages_whose_offsets_pass_32_bits(torch_dev, types, q_lens):
    """Pages 2^31 + 64 elements apart: append, then attention, as over pages
    side by side."""
    gh = _gh()
    b = P.batch(q_lens, [45, 9], heads=4, kv_heads=2, d=16, page=16, types=types, seed=30, spare=0, stale=0.0)
    x = P.to(b, torch_dev)
    num, far = x["k_pages"].shape[0], 2 ** 31 + 64
    room = torch.empty((num - 1) * far + 2 * 512, dtype=x["k_pages"].dtype, device=torch_dev)
    k, v = (room[at:].as_strided(x["k_pages"].shape, (far, 32, 16, 1)) for at in (0, 512))
    k.copy_(x["k_pages"])
    v.copy_(x["v_pages"])
    cos, sin = (t.to(torch_dev) for t in P.angles(x["page_table"].shape[1] * 16, 16))
    out = []
    for pages in ((x["k_pages"], x["v_pages"]), (k, v)):
        rest = (x["page_table"], x["q_offsets"], x["kv_lens"])
        q = gh.paged_append(*pages, *rest, x["k"], x["v"], q=x["q"], cos=cos, sin=sin)
        out.append(gh.paged_attention(q, *pages, *rest))
    assert torch.equal(k, x["k_pages"]) and torch.equal(v, x["v_pages"]) and torch.equal(*out)


@pytest.mark.parametrize("types", P.PAIRS, ids="/".join)
@pytest.mark.parametrize("count", [63, 64, 65, 300])
def test_many_sequences(torch_dev, types, count):
    q_lens = [(1, 0, 2, 1, 1)[i % 5] for i in range(count)]
    kv_lens = [(3, 17, 40, 1, 0)[(i * 7) % 5] + q_lens[i] for i in range(count)]
    for last in (1, 50):  # decode alone, and with a chunk
        q_lens[-1], kv_lens[-1] = last, last + 30
        b = P.batch(q_lens, kv_lens, heads=4, kv_heads=2, d=32, page=16, types=types, seed=31)
        _check(_attend(torch_dev, b), *P.attention(b))


@pytest.mark.parametrize("types", P.PAIRS, ids="/".join)
@pytest.mark.parametrize("count", [1, 64])
def test_a_wide_table_without_a_hint(torch_dev, types, count):
    """A table for a million positions and more of every sequence: the parts stay
    within what a stream keeps, the result the same."""
    gh = _gh()
    b = P.batch([1] * count, [40 + 13 * s for s in range(count)], heads=8, kv_heads=2, d=128, page=16, types=types, seed=33,
                width=1 << 17)
    x = P.to(b, torch_dev)
    assert gh.paged_attention_workspace_size(x["q"], *P.args(x)) <= 64 << 20
    _check(_attend(torch_dev, b), *P.attention(b))


def test_on_another_stream(torch_dev):
    gh = _gh()
    b = P.batch([1, 1, 60], [600, 33, 100], heads=8, kv_heads=2, d=64, page=16, types=("bf16", "bf16"), seed=32, stale=0.0)
    x = P.to(b, torch_dev)
    want = gh.paged_attention(x["q"], *P.args(x))
    streams = [torch.cuda.Stream() for _ in range(3)]
    out = []
    for s in streams:  # calls at once, each with its stream's workspace
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            out.append([gh.paged_attention(x["q"], *P.args(x)) for _ in range(5)])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for os in out for o in os)


# a value of the type next below 2, and a weight of about 1/2 that lies just under the
# middle between two of its values
@pytest.mark.parametrize("types", P.PAIRS, ids="/".join)
@pytest.mark.parametrize("lens", [([1], [30]), ([1], [900]), ([1] * 40, [4000] * 40), ([40], [900]), ([1, 300], [70, 1100])],
                         ids=lambda v: "-".join(map(str, (len(v[0]), v[0][-1]))))
def test_weights_add_up_to_what_the_product_sees(torch_dev, types, lens):
    """Where V is one value the result is that value: weights that are rounded for the
    product are rounded in their sum too.  Every 32nd key has weight 1, the others
    w.  Sums of n fp32 terms and a few more operations are off by (n + 16) 2^-24
    relatively, which is less than half a step of 16 bits, so those give the value
    itself."""
    h = P.half_step(P.TYPES[types[1]]) if types[1] != "f32" else 2.0 ** -8
    b = P.batch(*lens, heads=4, kv_heads=2, d=64, page=16, types=types, seed=50)
    value = 2 * (1 - h)
    b["q"].zero_()[..., 0] = 1
    for s, n in enumerate(lens[1]):
        at = torch.arange(n)
        page, row = b["page_table"][s, at // 16].long(), at % 16
        k = torch.zeros(n, 2, 64)
        k[..., 0] = -(at % 32 != 0).float()[:, None]
        b["k_pages"][page, row] = k.to(b["k_pages"].dtype)
        b["v_pages"][page, row] = value
    got = _attend(torch_dev, b, scale=-math.log(0.5 * (1 + h * (1 - 2 ** -4)))).double().cpu()
    if types[0] == "f32":
        assert (got - value).abs().max() <= (max(lens[1]) + 16) * 2.0 ** -24 * value
    else:
        assert (got == value).all(), (got - value).abs().max()


@pytest.mark.parametrize("types", P.PAIRS, ids="/".join)
@pytest.mark.parametrize("lens", [([1], [300]), ([1, 1], [5000, 40]), ([60], [300]), ([300, 1], [2000, 900])],
                         ids=lambda v: "-".join(map(str, v[0])))
@pytest.mark.parametrize("value", [float("inf"), float("-inf")])
def test_an_infinite_value_that_every_row_sees(torch_dev, types, lens, value):
    """It gives the rows what the formula has there, infinity of its sign, wherever
    its key lies; two of both signs give NaN."""
    b = P.batch(*lens, heads=4, kv_heads=2, d=64, page=16, types=types, seed=51)
    for at in (10, 129, 200):
        b["v_pages"][b["page_table"][0, at // 16].long(), at % 16, 1, at % 64] = value
    b["v_pages"][b["page_table"][0, 3].long(), 5, 0, 7] = value
    b["v_pages"][b["page_table"][0, 9].long(), 6, 0, 7] = -value
    want, bound = P.attention(b)
    got = _attend(torch_dev, b).double().cpu()
    for test in (torch.isposinf, torch.isneginf, torch.isnan):
        assert torch.equal(test(got), test(want)), test.__name__
    fine = torch.isfinite(want)
    assert (got - want).abs()[fine].le(bound[fine]).all()


@pytest.mark.parametrize("types", P.PAIRS, ids="/".join)
@pytest.mark.parametrize("lens", [([1], [300]), ([200], [300])], ids=lambda v: "-".join(map(str, v[0])))
def test_an_infinite_value_of_little_weight(torch_dev, types, lens):
    """2^-45 of the largest weight: nothing in f16, but not nothing."""
    b = P.batch(*lens, heads=4, kv_heads=2, d=64, page=16, types=types, seed=52)
    b["q"].zero_()[..., 0] = 1
    b["k_pages"][..., 0] = 0  # (rows without a position too)
    page = b["page_table"][0, 2].long()
    b["k_pages"][page, 3, :, 0] = -45
    b["v_pages"][page, 3, 0, 9] = float("inf")
    got = _attend(torch_dev, b, scale=math.log(2)).double().cpu()
    assert (got[:, :2, 9] == float("inf")).all()
    got[:, :2, 9] = 0
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("types", [("bf16", "bf16"), ("f32", "bf16"), ("f32", "f32")], ids="/".join)
@pytest.mark.parametrize("lens", [([1], [300]), ([1], [9000]), ([200], [300])], ids=lambda v: "-".join(map(str, v)))
def test_values_near_the_largest(torch_dev, types, lens):
    """V of 2^112 and more: sums of weights up to 1 times V stay finite, whatever
    constant the weights carry on the way."""
    b = P.batch(*lens, heads=4, kv_heads=2, d=64, page=16, types=types, seed=53)
    b["v_pages"] *= 2.0 ** 112
    _check(_attend(torch_dev, b), *P.attention(b))


@pytest.mark.parametrize("types", [("bf16", "bf16"), ("f32", "bf16"), ("f32", "f32")], ids="/".join)
def test_values_near_the_largest_under_a_late_maximum(torch_dev, types):
    """Scores that rise by less than what the running maximum may lag: weights of up
    to 2^7.5 before V of 2^118."""
    b = P.batch([520], [700], d=32, types=types, seed=56, **MANY)
    b["q"].zero_()[..., 0] = 1
    at = torch.arange(700)
    page, row = b["page_table"][0, at // 24].long(), at % 24
    k = torch.zeros(700, 32, 32)
    k[64:, :, 0] = 7.5
    b["k_pages"][page, row] = k.to(b["k_pages"].dtype)
    b["v_pages"][page, row] = 2.0 ** 118
    want, bound = P.attention(b, scale=math.log(2))
    _check(_attend(torch_dev, b, scale=math.log(2))[:520], want[:520], bound[:520])


@pytest.mark.parametrize("types", P.PAIRS, ids="/".join)
@pytest.mark.parametrize("lens", [([1], [1000]), ([30], [1000]), ([200], [1000])], ids=lambda v: "-".join(map(str, v[0])))
@pytest.mark.parametrize("page", [8, 16, 24])
def test_pages_before_the_window_may_be_gone(torch_dev, types, lens, page):
    """Pages none of whose keys any new token sees are not asked for: status stays."""
    gh = _gh()
    window = 100
    b = P.batch(*lens, heads=4, kv_heads=2, d=64, page=page, types=types, seed=54)
    want = P.attention(b, window=window)
    first = lens[1][0] - lens[0][0] + 1 - window
    b["page_table"][0, :first // page] = -1
    x = P.to(b, torch_dev)
    st = torch.zeros(1, dtype=torch.int32, device=torch_dev)
    got = gh.paged_attention(x["q"], *P.args(x), window=window, status=st)
    _check(got, *want)
    assert int(st) == 0


@pytest.mark.parametrize("types", P.PAIRS, ids="/".join)
@pytest.mark.parametrize("lens", [([2], [1]), ([1, 3, 1], [4, 2, 9]), ([1, 200, 1], [5, 199, 70])],
                         ids=lambda v: "-".join(map(str, v[0])))
def test_tokens_before_position_0_are_reported(torch_dev, types, lens):
    """More new tokens than positions: the attention says so as the append does."""
    gh = _gh()
    b = P.batch(*lens, heads=4, kv_heads=2, d=64, page=16, types=types, seed=55)
    x = P.to(b, torch_dev)
    st = torch.zeros(1, dtype=torch.int32, device=torch_dev)
    _check(gh.paged_attention(x["q"], *P.args(x), status=st), *P.attention(b))
    assert int(st) == 1
    st.zero_()
    gh.paged_append(*P.args(x), x["k"], x["v"], status=st)
    assert int(st) == 1


# more than 1024 pages in one workgroup's keys, which takes those in turn (a small
# hint keeps the axis whole): pages of 1 and 3 positions, pages of 16 past 16384 keys.
# A window begins inside a page, so that such a turn ends inside a tile.
@pytest.mark.parametrize("types", P.PAIRS, ids="/".join)
@pytest.mark.parametrize("q_lens,kv_lens,page,window", [
    ([1], [3000], 1, 0), ([1, 1], [5000, 1030], 3, 0), ([1], [5000], 3, 4001), ([2], [3500], 1, 2777),
    ([1], [17500], 16, 0), ([1], [18000], 16, 16999), ([150], [3300], 1, 0), ([200, 1], [5000, 3200], 3, 0),
    ([200], [5000], 3, 3333), ([140], [17001], 16, 0), ([140], [17001], 16, 16500),
], ids=str)
def test_more_pages_than_are_looked_up_at_once(torch_dev, types, q_lens, kv_lens, page, window):
    b = P.batch(q_lens, kv_lens, heads=4, kv_heads=2, d=64, page=page, types=types, seed=57)
    _check(_attend(torch_dev, b, window=window, max_kv_len=100), *P.attention(b, window=window))


@pytest.mark.parametrize("types", P.PAIRS, ids="/".join)
@pytest.mark.parametrize("page,kv,window", [(1, 2500, 0), (3, 4000, 0), (3, 4000, 3301)])
def test_more_pages_than_are_looked_up_at_once_of_many_heads(torch_dev, types, page, kv, window):
    b = P.batch([520], [kv], d=32, heads=32, kv_heads=32, page=page, types=types, seed=58)
    _check(_attend(torch_dev, b, window=window, max_kv_len=100), *P.attention(b, window=window))


@pytest.mark.parametrize("types", P.PAIRS, ids="/".join)
@pytest.mark.parametrize("q_len,page,kv", [(1, 1, 3000), (4, 3, 4000), (150, 1, 3300), (200, 3, 5000)])
def test_infinite_values_past_the_pages_looked_up_first(torch_dev, types, q_len, page, kv):
    """One that every token sees, one that only the last does."""
    b = P.batch([q_len], [kv], heads=4, kv_heads=2, d=64, page=page, types=types, seed=59)
    for at, dim in ((kv - 400, 3), (kv - 1, 5)):
        b["v_pages"][b["page_table"][0, at // page].long(), at % page, 1, dim] = float("inf")
    want, bound = P.attention(b)
    got = _attend(torch_dev, b, max_kv_len=100).double().cpu()
    assert torch.equal(torch.isposinf(got), torch.isposinf(want)) and not torch.isnan(got).any()
    fine = torch.isfinite(want)
    assert (got - want).abs()[fine].le(bound[fine]).all()


@pytest.mark.parametrize("types", [("bf16", "bf16"), ("f16", "f16")], ids="/".join)
@pytest.mark.parametrize("lens", [([1], [300]), ([1], [5000]), ([1] * 6, [33, 1, 700, 64, 129, 2000]), ([3, 0, 1, 4], [50, 40, 65, 300])],
                         ids=lambda v: "-".join(map(str, v[0])))
def test_single_tokens_lose_nothing_to_the_weights(torch_dev, types, lens):
    """As _paged's bound, but for the weights' rounding: two pieces leave half a step
    of half a step."""
    h = P.half_step(P.TYPES[types[0]])
    for heads, kv_heads, d in ((8, 2, 128), (4, 4, 64)):
        b = P.batch(*lens, heads=heads, kv_heads=kv_heads, d=d, page=16, types=types, seed=61)
        want, bound = P.attention(b)
        size = P.attention(dict(b, v_pages=b["v_pages"].abs()))[0]
        _check(_attend(torch_dev, b), want, bound - size * (h - h * h))


@pytest.mark.parametrize("types", P.PAIRS, ids="/".join)
@pytest.mark.parametrize("lens", [([1], [300]), ([3], [4000]), ([60], [300]), ([300], [500])],
                         ids=lambda v: "-".join(map(str, v)))
@pytest.mark.parametrize("d", [24, 64, 128])
def test_rows_one_by_one_over_a_page_outside_the_cache(torch_dev, types, lens, d):
    """A NaN that only the last token sees sends its workgroup's rows through their
    keys one by one; the pages outside the cache read as zeros there too."""
    gh = _gh()
    b = P.batch(*lens, heads=4, kv_heads=2, d=d, page=16, types=types, seed=62, spare=5)
    n = lens[1][0]
    where = b["page_table"][0, (n - 1) // 16].long(), (n - 1) % 16, 1, 2
    b["v_pages"][where] = float("nan")
    unused = sorted(set(range(b["k_pages"].shape[0])) - set(b["page_table"].flatten().tolist()))[0]
    for pages in ("k_pages", "v_pages"):
        b[pages][unused] = 0
    bad = dict(b, page_table=b["page_table"].clone())
    for at in (0, 7, 8, 9, 10, 16):
        b["page_table"][0, at] = unused
        bad["page_table"][0, at] = -1 if at % 2 else 10 ** 6
    want, bound = P.attention(b)
    x = P.to(bad, torch_dev)
    got = gh.paged_attention(x["q"], *P.args(x)).double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.isnan(got[-1, 2:, 2]).all()
    fine = torch.isfinite(want)
    assert (got - want).abs()[fine].le(bound[fine]).all()


@pytest.mark.parametrize("types", [t for t in P.PAIRS if t[0] != "f16"], ids="/".join)
def test_attention_scale_of_nothing_over_huge_scores(torch_dev, types):
    """All weights are equal where the scale is 0, however large the products."""
    b = P.batch([1, 60, 400], [200, 150, 900], heads=4, kv_heads=2, d=64, page=16, types=types, seed=41)
    b["q"] *= 1e36
    _check(_attend(torch_dev, b, scale=0.0), *P.attention(b, scale=0.0))
    _check(_attend(torch_dev, b, scale=0.0, window=40), *P.attention(b, scale=0.0, window=40))
