"""A ragged batch over a paged cache for the tests, its plain form in 64 bits
and the bounds that rounding gives."""
import math

import torch

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
PAIRS = [("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"), ("f32", "bf16")]


def half_step(dtype):
    """The largest relative error of one rounding."""
    return torch.finfo(dtype).eps / 2


def batch(q_lens, kv_lens, *, heads, kv_heads, d, page, types=("f32", "f32"), seed=0, pad=0, spare=3, width=None,
          stale=float("nan"), layout="rows"):
    """Tensors on the CPU.  Rows of the pages that hold no position are
    `stale`; `pad` rows of tokens lie behind the last sequence.  layout "rows":
    [pages, page, kv_heads, d]; "heads": the same from [pages, kv_heads, page,
    d] memory; "pairs": K and V side by side in one tensor."""
    g = torch.Generator().manual_seed(seed)
    ta, tc = TYPES[types[0]], TYPES[types[1]]
    pages = [-(-n // page) for n in kv_lens]
    total = sum(pages) + spare
    order = torch.randperm(total, generator=g)
    width = max(pages + [1]) if width is None else width
    table = torch.full((len(q_lens), width), -1, dtype=torch.int32)
    at = 0
    for s, n in enumerate(pages):
        table[s, :n] = order[at:at + n].to(torch.int32)
        at += n
    if layout == "pairs":
        both = torch.full((total, 2, page, kv_heads, d), stale, dtype=tc)
        k, v = both[:, 0], both[:, 1]
    elif layout == "heads":
        k, v = (torch.full((total, kv_heads, page, d), stale, dtype=tc).transpose(1, 2) for _ in range(2))
    else:
        k, v = (torch.full((total, page, kv_heads, d), stale, dtype=tc) for _ in range(2))
    for s, n in enumerate(kv_lens):
        for p in range(pages[s]):
            rows = min(page, n - p * page)
            k[table[s, p], :rows] = torch.randn(rows, kv_heads, d, generator=g).to(tc)
            v[table[s, p], :rows] = torch.randn(rows, kv_heads, d, generator=g).to(tc)
    tokens = sum(q_lens) + pad
    mk = lambda h: torch.randn(tokens, h, d, generator=g).to(ta)  # noqa: E731
    return {"q": mk(heads), "k": mk(kv_heads), "v": mk(kv_heads), "k_pages": k, "v_pages": v, "page_table": table,
            "q_offsets": torch.tensor([0] + q_lens).cumsum(0).to(torch.int32),
            "kv_lens": torch.tensor(kv_lens, dtype=torch.int32), "page": page, "tokens": tokens}


def rows_of(b, s):
    """K and V of sequence s, [kv_len, kv_heads, d] in 64 bits."""
    n, page = int(b["kv_lens"][s]), b["page"]
    at = b["page_table"][s, :-(-n // page)].long()
    return tuple(b[t][at].flatten(0, 1)[:n].double() for t in ("k_pages", "v_pages"))


def attention(b, *, scale=None, causal=True, window=0):
    """(out, bound) in 64 bits; rows of no sequence are NaN.  The bound counts
    the roundings: scores are dot products of d terms and a few more fp32
    operations (delta, their absolute error, moves a probability by as much
    relatively), exp2 is good to 2^-22, P is rounded to the 16-bit type (fp32:
    2^-24), sums of n terms in fp32, and the result is rounded once."""
    tokens, heads, d = b["q"].shape
    out = torch.full((tokens, heads, d), float("nan"), dtype=torch.float64)
    bound = torch.zeros(tokens, heads, d, dtype=torch.float64)
    scale = 1 / math.sqrt(d) if scale is None else scale
    u, h = 2.0 ** -24, half_step(b["q"].dtype)
    for s in range(len(b["kv_lens"])):
        k, v = rows_of(b, s)
        n = k.shape[0]
        g = heads // k.shape[1]
        a, e = int(b["q_offsets"][s]), int(b["q_offsets"][s + 1])
        for t in range(a, e):
            p = n - (e - t)
            lo = max(0, p - window + 1) if window else 0
            hi = min(n, p + 1) if causal else n
            if hi <= lo:
                out[t] = 0
                continue
            kk, vv = (x[lo:hi].repeat_interleave(g, 1) for x in (k, v))  # [n, heads, d]
            q = b["q"][t].double()
            w = torch.einsum("hd,nhd->hn", q, kk) * scale
            prob = torch.softmax(w, -1)
            out[t] = torch.einsum("hn,nhd->hd", prob, vv)
            size = torch.einsum("hn,nhd->hd", prob, vv.abs())
            delta = u * (d + 8) * abs(scale) * torch.einsum("hd,nhd->hn", q.abs(), kk.abs()).amax(-1, keepdim=True)
            bound[t] = h * out[t].abs() + size * (h + 2 * delta + 2.0 ** -21 + (hi - lo) * u)
    return out, bound


def turned(x, pos, cos, sin, interleaved):
    """x [heads, d] at a position, in 64 bits."""
    y = x.double().clone()
    if cos is None:
        return y
    half = cos.shape[1]
    c, s = cos[pos].double(), sin[pos].double()
    i = torch.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    y[:, a], y[:, b] = x.double()[:, a] * c - x.double()[:, b] * s, x.double()[:, b] * c + x.double()[:, a] * s
    return y


def angles(rows, rotary_dim, base=10000.0):
    f = base ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    a = torch.arange(rows, dtype=torch.float64)[:, None] * f
    return a.cos().float(), a.sin().float()


def to(b, dev):
    """The batch on the device, with the same strides."""
    out = {}
    both = None
    for n, t in b.items():
        if not torch.is_tensor(t):
            out[n] = t
            continue
        if n in ("k_pages", "v_pages"):
            base = t._base if t._base is not None else t
            if base.dim() == 5:  # K and V in one tensor
                both = base.to(dev) if both is None else both
                out[n] = both[:, 0 if n == "k_pages" else 1]
            elif base is not t:
                out[n] = base.to(dev).transpose(1, 2)
            else:
                out[n] = t.to(dev)
        else:
            out[n] = t.to(dev)
    return out


def args(b):
    return b["k_pages"], b["v_pages"], b["page_table"], b["q_offsets"], b["kv_lens"]
