"""PagedKVCache, MultiHeadAttention.step_paged and the 4-bit layers: the
bookkeeping on the CPU, and whole steps on the GPU against the same steps in
64 bits."""
import math

import pytest
import torch

import _paged as P


def _gh():
    import ghostflow_hip as gh

    return gh


def _cache(pages=10, page=4, heads=2, d=8, **kw):
    return _gh().PagedKVCache(pages, page, heads, d, **kw)


# ---- bookkeeping -------------------------------------------------------------------

def test_pages_grow_and_come_back():
    c = _cache(device="cpu")
    a, b = c.add(), c.add()
    first = c.extend([a, b], [5, 1])
    assert first.tokens == 6 and first.max_kv_len == 5 and c.free_pages == 7
    assert first.q_offsets.tolist() == [0, 5, 6] and first.kv_lens.tolist() == [5, 1]
    assert first.page_table.shape == (2, 2) and first.page_table[1, 1] == -1
    second = c.extend([b, a], [4, 3])  # a fills its pages, b takes one more
    assert c.length(a) == 8 and c.length(b) == 5 and c.free_pages == 6
    assert second.page_table[1].tolist() == first.page_table[0].tolist()
    used = second.page_table.flatten().tolist()
    assert len(set(used)) == 4 and min(used) >= 0
    c.remove(a)
    assert c.free_pages == 8
    d = c.add()
    assert c.extend([d], [0]).page_table.tolist() == [[-1]] and c.extend([d], [32]).max_kv_len == 32
    assert c.free_pages == 0


def test_an_empty_batch():
    b = _cache(device="cpu").extend([], [])
    assert b.tokens == 0 and b.max_kv_len == 0 and b.q_offsets.tolist() == [0] and b.page_table.shape == (0, 1)


def test_refusals_change_nothing():
    gh = _gh()
    c = _cache(pages=3, device="cpu")
    a, b = c.add(), c.add()
    c.extend([a], [4])
    for seqs, counts in (([a, a], [1, 1]), ([a, b], [1]), ([a], [-1]), ([7], [1]), ([a, b], [4, 5])):
        with pytest.raises(gh.GhostFlowError):
            c.extend(seqs, counts)
        assert c.free_pages == 2 and c.length(a) == 4 and c.length(b) == 0
    c.remove(a)
    with pytest.raises(gh.GhostFlowError):
        c.remove(a)
    for bad in ((0, 4, 2, 8), (3, 0, 2, 8), (3, 4, 0, 8), (3, 4, 2, 0)):
        with pytest.raises(gh.GhostFlowError):
            gh.PagedKVCache(*bad, device="cpu")


def test_step_refuses_rows_that_are_not_the_batch():
    gh = _gh()
    c = _cache(device="cpu")
    m = gh.MultiHeadAttention(16, 2, device="cpu")
    m.eval()
    batch = c.extend([c.add()], [3])
    for shape in ((2, 16), (3, 8), (1, 3, 16)):
        with pytest.raises(gh.GhostFlowError):
            m.step_paged(torch.zeros(shape), c, batch)


# ---- whole steps -------------------------------------------------------------------

class Plain:
    """The layer in 64 bits over whole sequences."""

    def __init__(self, weights, heads, cos=None, sin=None):
        self.w = [w.double().cpu() for w in weights]
        self.heads, self.cos, self.sin = heads, cos, sin

    def attend(self, x, lens, window=0):
        """x: all tokens so far of every sequence; the outputs of the last
        lens[i] of each."""
        out = []
        for t, n in zip(x, lens):
            t = t.double()
            q, k, v = ((t @ self.w[2 * i].t() + self.w[2 * i + 1]).view(len(t), self.heads, -1) for i in range(3))
            if self.cos is not None:
                q, k = (torch.stack([P.turned(r, p, self.cos, self.sin, False) for p, r in enumerate(y)]) for y in (q, k))
            at = torch.arange(len(t))
            s = torch.einsum("qhd,khd->hqk", q, k) / math.sqrt(q.shape[-1])
            sees = (at[None] <= at[:, None]) & ((at[None] > at[:, None] - window) | (window == 0))
            y = torch.einsum("hqk,khd->qhd", torch.softmax(s.masked_fill(~sees, -math.inf), -1), v)
            out.append((y.flatten(1) @ self.w[6].t() + self.w[7])[len(t) - n:])
        return torch.cat(out)


@pytest.mark.gpu
@pytest.mark.parametrize("quantized", [False, True])
@pytest.mark.parametrize("rotary", [False, True])
@pytest.mark.parametrize("window", [0, 9])
def test_steps_of_a_ragged_batch(torch_dev, quantized, rotary, window):
    """Prompts in chunks, single tokens, a sequence that leaves and one that
    takes its pages, fp32: every step is the layer over the whole sequence.
    1e-4 of the largest output covers some hundred roundings of 2^-24 of
    sums that are at most a few hundred times the outputs."""
    gh = _gh()
    torch.manual_seed(3)
    e, heads = 64, 4
    m = gh.MultiHeadAttention(e, heads)
    m.eval()
    weights = m.parameters()
    if quantized:
        m.quantize_grouped(32, symmetric=False)
        weights = [t for w in m.w4 for t in (w.dequantize(), w.bias)]
    cos, sin = P.angles(80, e // heads) if rotary else (None, None)
    dev = [None if t is None else t.to(torch_dev) for t in (cos, sin)]
    plain = Plain(weights, heads, cos, sin)
    c = gh.PagedKVCache(14, 5, heads, e // heads)
    seqs = {c.add(): torch.empty(0, e) for _ in range(3)}
    ids = list(seqs)

    def step(which, counts):
        new = [torch.randn(n, e) for n in counts]
        for s, t in zip(which, new):
            seqs[s] = torch.cat((seqs[s], t))
        got = m.step_paged(torch.cat(new).to(torch_dev), c, c.extend(which, counts), cos=dev[0], sin=dev[1], window=window)
        want = plain.attend([seqs[s] for s in which], counts, window)
        assert (got.cpu().double() - want).abs().max() <= 1e-4 * want.abs().max()

    step(ids, [17, 1, 8])
    step(ids, [1, 1, 1])
    step([ids[2], ids[0]], [6, 1])
    step(ids, [1, 3, 0])
    c.remove(ids[0])
    late = c.add()
    seqs[late] = torch.empty(0, e)
    step([ids[1], late, ids[2]], [1, 20, 1])
    step([late, ids[1], ids[2]], [1, 1, 1])


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_a_decode_step_of_16_bits(torch_dev, kind):
    """4-bit projections, append, attention and projection back on 16-bit
    activations over a cache of the same type.  Four roundings to the type
    follow each other (q, k, v; P; the attention; the result), each of half a
    step relative to sums of magnitudes that exceed the result's largest by
    less than 16 here."""
    gh = _gh()
    torch.manual_seed(4)
    e, heads, dt = 256, 4, P.TYPES[kind]
    m = gh.MultiHeadAttention(e, heads)
    m.eval()
    m.quantize_grouped(64)
    plain = Plain([t for w in m.w4 for t in (w.dequantize(), w.bias)], heads)
    c = gh.PagedKVCache(40, 16, heads, e // heads, dtype=dt)
    ids = [c.add() for _ in range(4)]
    xs = [(torch.randn(n, e) * 0.3).to(dt) for n in (40, 3, 100, 1)]
    m.step_paged(torch.cat(xs).to(torch_dev), c, c.extend(ids, [len(x) for x in xs]))
    new = (torch.randn(4, e) * 0.3).to(dt)
    got = m.step_paged(new.to(torch_dev), c, c.extend(ids, [1] * 4))
    assert got.dtype == dt
    want = plain.attend([torch.cat((x, t[None])) for x, t in zip(xs, new)], [1] * 4)
    assert (got.cpu().double() - want).abs().max() <= 4 * 16 * P.half_step(dt) * want.abs().max()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 3, 40])
def test_swiglu_on_4_bit_weights(torch_dev, rows):
    gh = _gh()
    torch.manual_seed(5)
    layer = gh.SwiGLU(96, 160)
    q = layer.quantize_grouped(32)
    x = torch.randn(2, rows, 96)
    w = [(p.dequantize().double().cpu(), p.bias.double().cpu()) for p in (q.gate, q.up, q.down)]
    g, u = (x.double() @ w[i][0].t() + w[i][1] for i in range(2))
    want = (g / (1 + torch.exp(-g)) * u) @ w[2][0].t() + w[2][1]
    got = q(x.to(torch_dev)).cpu().double()
    # sums of 96 and 160 terms, a few fp32 operations between
    assert got.shape == want.shape and (got - want).abs().max() <= 300 * 2.0 ** -24 * 16 * want.abs().max()
    assert q.gate.compression_ratio() == 32 * 4 / (32 / 2 + 4)  # a group: fp32, then codes and a scale
    with pytest.raises(gh.GhostFlowError):
        q(x.to(torch_dev)[..., :64])
