"""Performance cases of the decode-step operators: what a serving program
calls for every layer and step, over the ranges it is used in.

  append      rotary positions applied to q and k, and k / v written into the
              pages of a ragged batch of sequences
  attention   that batch's new tokens (one each, or chunks of a prompt) over
              the pages: causal, with an optional window, grouped heads
  linear_w4   Linear on 4-bit weights with group scales
  quantize_w4 a weight to 4 bits in groups and back, as quantization-aware
              training and the loader of a model do

A ragged batch is `page_table` [seqs, pages], `q_offsets` [seqs + 1] (rows of
the new tokens) and `kv_lens` [seqs] (positions including the new ones).

`listed()` names some, `draw()` gives others from the same ranges.  Inputs are
made on the GPU from the seed alone.
"""
import math
import os
import random
import sys

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}


def _gh():
    pkg = os.path.join(os.getcwd(), "ghost-flow_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import ghostflow_hip
    return ghostflow_hip


def listed():
    return [
        # one decode step of 64 sequences: a few tokens, latency of the step
        {"name": "append_decode_64", "kind": "append", "type": "bf16", "cache": "bf16", "h": 32, "hkv": 8, "d": 128,
         "seqs": 64, "q": 1, "kv": 4096, "page": 16, "rot": 128, "inter": False},
        # four long prompts, fp32 activations into a 16-bit cache
        {"name": "append_prompts", "kind": "append", "type": "f32", "cache": "bf16", "h": 32, "hkv": 8, "d": 128,
         "seqs": 4, "q": 4000, "kv": 4000, "page": 64, "rot": 128, "inter": False},
        # a single user's next token, small heads: latency
        {"name": "attn_decode_1_f16", "kind": "attention", "type": "f16", "cache": "f16", "h": 12, "hkv": 12, "d": 64,
         "seqs": 1, "q": 1, "kv": 517, "page": 16, "window": 0},
        # the decode step of a loaded server
        {"name": "attn_decode_64_bf16", "kind": "attention", "type": "bf16", "cache": "bf16", "h": 32, "hkv": 8,
         "d": 128, "seqs": 64, "q": 1, "kv": 4096, "page": 16, "window": 0},
        # the framework's own head layout and type: 4 sequences, fp32, no groups
        {"name": "attn_decode_4_f32", "kind": "attention", "type": "f32", "cache": "f32", "h": 32, "hkv": 32,
         "d": 128, "seqs": 4, "q": 1, "kv": 2047, "page": 64, "window": 0},
        # chunks of several prompts beside sequences that decode, fp32 over a
        # 16-bit cache, with a window
        {"name": "attn_mixed_f32_bf16", "kind": "attention", "type": "f32", "cache": "bf16", "h": 32, "hkv": 8,
         "d": 128, "seqs": 6, "q": 700, "kv": 3000, "page": 16, "window": 1024},
        # a chunk of a long prompt
        {"name": "attn_chunk_2048_bf16", "kind": "attention", "type": "bf16", "cache": "bf16", "h": 32, "hkv": 8,
         "d": 128, "seqs": 1, "q": 2048, "kv": 16384, "page": 64, "window": 0},
        # one token through a 4096-wide projection
        {"name": "w4_m1_f32", "kind": "linear_w4", "type": "f32", "m": 1, "k": 4096, "n": 4096, "group": 128,
         "zeros": False, "bias": True},
        # 16 sequences through a down projection, with zero points
        {"name": "w4_m16_bf16", "kind": "linear_w4", "type": "bf16", "m": 16, "k": 14336, "n": 4096, "group": 64,
         "zeros": True, "bias": False},
        # 50 rows through an up projection
        {"name": "w4_m50_f16", "kind": "linear_w4", "type": "f16", "m": 50, "k": 4096, "n": 11008, "group": 128,
         "zeros": False, "bias": False},
        # a projection's weight, symmetric
        {"name": "q4_4096", "kind": "quantize_w4", "n": 4096, "k": 4096, "group": 128, "zeros": False},
        # an odd number of rows in small groups with zero points
        {"name": "q4_1001_zeros", "kind": "quantize_w4", "n": 1001, "k": 11008, "group": 32, "zeros": True},
    ]


# ---- drawing more cases of the same ranges ------------------------------------


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    return rng.choice(((32, 8, 128), (32, 32, 128), (12, 12, 64), (16, 4, 64), (8, 1, 128), (28, 4, 128), (20, 5, 80),
                       (16, 2, 96)))


def _types(rng):
    return rng.choice((("bf16", "bf16"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "f32"), ("f32", "bf16")))


def draw(rng):
    while True:
        c = _draw(rng)
        if c["kind"] == "attention" and 4 * c["seqs"] * c["h"] * c["q"] * c["kv"] > 5e9:
            continue  # scores of the plain form
        if "kv" in c and c["seqs"] * c["kv"] * c["hkv"] * c["d"] > 5e8:
            continue  # pages
        w = work(c)
        if w["flops"] <= 5e11 and w["bytes"] <= 6.5e8:
            return c


def _draw(rng):
    kind = rng.choice(("append", "attention", "attention", "linear_w4", "linear_w4", "quantize_w4"))
    if kind in ("append", "attention"):
        (h, hkv, d), (t, cache) = _heads(rng), _types(rng)
        seqs = _log(rng, 1, 64)
        q = 1 if rng.random() < 0.5 else _log(rng, 2, 4000 if kind == "append" else 2048)
        c = {"kind": kind, "type": t, "cache": cache, "h": h, "hkv": hkv, "d": d, "seqs": seqs, "q": q,
             "kv": max(q, _log(rng, 64, 16384)), "page": rng.choice((16, 16, 32, 64, 128))}
        if kind == "append":
            c.update(rot=rng.choice((d, d, d // 2)), inter=rng.random() < 0.3)
        else:
            c.update(window=0 if rng.random() < 0.6 else _log(rng, 100, 4096))
        return c
    group = rng.choice((32, 64, 128, 128))
    c = {"kind": kind, "k": _log(rng, 512 // 32, 14336 // 32) * 32, "group": group, "zeros": rng.random() < 0.5}
    if kind == "linear_w4":
        c.update(n=_log(rng, 512, 14336), type=rng.choice(("f32", "bf16", "f16")), m=_log(rng, 1, 64),
                 bias=rng.random() < 0.4)
    else:
        c["n"] = _log(rng, 512, 8192)
    return c


# ---- what a program has in hand -------------------------------------------------


def _lens(c):
    """New tokens and positions of every sequence: the first has the most, the
    others between a quarter and all of it, every third of a batch of chunks a
    single token."""
    r = random.Random(c["seqs"] * 1000003 + c["kv"] * 1009 + c["q"])
    ql, kl = [], []
    for s in range(c["seqs"]):
        q = c["q"] if s == 0 else 1 if s % 3 == 2 else r.randint(max(1, c["q"] // 4), c["q"])
        kv = c["kv"] if s == 0 else r.randint(max(1, c["kv"] // 4), c["kv"])
        ql.append(q)
        kl.append(max(q, kv))
    return ql, kl


def _batch(c, g, s):
    ql, kl = _lens(c)
    pages = [-(-n // c["page"]) for n in kl]
    total, width = sum(pages), max(pages)
    # the pool is larger than the batch, and a sequence's pages lie anywhere
    order = torch.randperm(total + total // 8 + 3, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(c["seqs"], width, dtype=torch.int32, device="cuda")
    at = torch.tensor([0] + pages, device="cuda").cumsum(0)
    col = torch.arange(width, device="cuda")
    used = col < torch.tensor(pages, device="cuda")[:, None]
    table[used] = order[(at[:-1, None] + col)[used]]
    s["page_table"] = table
    s["q_offsets"] = torch.tensor([0] + ql, device="cuda").cumsum(0).to(torch.int32)
    s["kv_lens"] = torch.tensor(kl, dtype=torch.int32, device="cuda")
    s["max_q"], s["max_kv"], s["tokens"] = max(ql), max(kl), sum(ql)
    t = _TYPES[c["cache"]]
    shape = (order.numel(), c["page"], c["hkv"], c["d"])
    # (whole pages hold something: what earlier sequences left there)
    s["k_pages"] = torch.randn(shape, generator=g, device="cuda").to(t)
    s["v_pages"] = torch.randn(shape, generator=g, device="cuda").to(t)


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))

    def normal(*shape, t="f32", std=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(_TYPES[t])

    s = dict(c)
    if c["kind"] in ("append", "attention"):
        _batch(c, g, s)
        s["q"] = normal(s["tokens"], c["h"], c["d"], t=c["type"])
        s["out"] = torch.zeros_like(s["q"])
    if c["kind"] == "append":
        s["k"] = normal(s["tokens"], c["hkv"], c["d"], t=c["type"])
        s["v"] = normal(s["tokens"], c["hkv"], c["d"], t=c["type"])
        rows = s["page_table"].shape[1] * c["page"]
        freq = 10000.0 ** (-torch.arange(0, c["rot"], 2, dtype=torch.float64, device="cuda") / c["rot"])
        angle = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * freq
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    elif c["kind"] == "linear_w4":
        s["x"] = normal(c["m"], c["k"], t=c["type"])
        s["codes"] = torch.randint(0, 256, (c["n"], c["k"] // 2), dtype=torch.uint8, generator=g, device="cuda")
        groups = -(-c["k"] // c["group"])
        s["scales"] = (0.5 + torch.rand(c["n"], groups, generator=g, device="cuda")) * (0.2 / math.sqrt(c["k"]))
        s["zero_points"] = (torch.randint(4, 12, (c["n"], groups), dtype=torch.uint8, generator=g, device="cuda")
                            if c["zeros"] else None)
        s["b"] = normal(c["n"], t=c["type"], std=0.1) if c["bias"] else None
    elif c["kind"] == "quantize_w4":
        s["w"] = normal(c["n"], c["k"], std=0.02)
    return s


# ---- one pass -------------------------------------------------------------------


def run(state):
    s = state
    if own:
        gh = _gh()
        if s["kind"] == "append":
            gh.paged_append(s["k_pages"], s["v_pages"], s["page_table"], s["q_offsets"], s["kv_lens"], s["k"], s["v"],
                            q=s["q"], q_out=s["out"], cos=s["cos"], sin=s["sin"], interleaved=s["inter"])
            return s["out"], s["k_pages"], s["v_pages"]
        if s["kind"] == "attention":
            return gh.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["page_table"], s["q_offsets"],
                                      s["kv_lens"], causal=True, window=s["window"], max_kv_len=s["max_kv"],
                                      out=s["out"])
        if s["kind"] == "linear_w4":
            return gh.linear_w4(s["x"], s["codes"], s["scales"], s["zero_points"], s["b"], group_size=s["group"])
        codes, scales, zeros = gh.quantize_grouped_i4(s["w"], s["group"], symmetric=not s["zeros"])
        return gh.dequantize_grouped_i4(codes, scales, zeros, s["group"]), scales, zeros
    return {"append": _append, "attention": _attention, "linear_w4": _linear_w4, "quantize_w4": _quantize_w4}[s["kind"]](s)


def _rows_of(s):
    """Sequence and position of every new token."""
    t = torch.arange(s["tokens"], device="cuda")
    off = s["q_offsets"].long()
    seq = torch.bucketize(t, off[1:], right=True)
    return seq, s["kv_lens"].long()[seq] - off[seq + 1] + t


def _rotate(x, c, s, rot, inter):
    x = x.float()
    c, s = c[:, None], s[:, None]
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if inter else (x[..., :rot // 2], x[..., rot // 2:rot])
    p, q = a * c - b * s, b * c + a * s
    y = torch.stack((p, q), -1).flatten(-2) if inter else torch.cat((p, q), -1)
    return torch.cat((y, x[..., rot:]), -1)


def _append(s):
    seq, pos = _rows_of(s)
    c, sn = s["cos"][pos], s["sin"][pos]
    page, row = s["page_table"][seq, pos // s["page"]].long(), pos % s["page"]
    t = s["k_pages"].dtype
    s["out"].copy_(_rotate(s["q"], c, sn, s["rot"], s["inter"]))
    s["k_pages"][page, row] = _rotate(s["k"], c, sn, s["rot"], s["inter"]).to(t)
    s["v_pages"][page, row] = s["v"].to(t)
    return s["out"], s["k_pages"], s["v_pages"]


def _attention(s):
    # every sequence padded to the longest
    nq, nk, h, hkv, d = s["max_q"], s["max_kv"], s["h"], s["hkv"], s["d"]
    j = torch.arange(nk, device="cuda")
    page, row = s["page_table"][:, j // s["page"]].long(), j % s["page"]
    k = s["k_pages"][page, row].float().permute(0, 2, 3, 1).contiguous()  # [S, hkv, d, nk]
    v = s["v_pages"][page, row].float().transpose(1, 2).contiguous()      # [S, hkv, nk, d]
    off, kl = s["q_offsets"].long(), s["kv_lens"].long()
    i = torch.arange(nq, device="cuda")
    ql = off[1:] - off[:-1]
    q = s["q"][(off[:-1, None] + i).clamp(max=s["tokens"] - 1)].float()   # [S, nq, h, d]
    q = q.view(-1, nq, hkv, h // hkv, d).permute(0, 2, 3, 1, 4).reshape(-1, hkv, h // hkv * nq, d)
    score = (torch.matmul(q, k) * (1.0 / math.sqrt(d))).view(-1, hkv, h // hkv, nq, nk)
    pos = (kl - ql)[:, None] + i
    keep = j <= pos[..., None]
    if s["window"]:
        keep = keep & (j > pos[..., None] - s["window"])
    score = score.masked_fill_(~keep[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(-1, hkv, h // hkv * nq, nk), v).view(-1, hkv, h // hkv, nq, d)
    o = (o / torch.where(total == 0, 1.0, total)).permute(0, 3, 1, 2, 4).reshape(-1, nq, h, d)
    live = i < ql[:, None]
    s["out"][:] = o[live].to(s["out"].dtype)
    return s["out"]


def _codes(packed):
    return torch.stack((packed & 15, packed >> 4), -1).flatten(1)


def _spread(v, k, group):
    """One value per group to one per column."""
    return v.repeat_interleave(group, 1)[:, :k]


def _linear_w4(s):
    zero = 8.0 if s["zero_points"] is None else _spread(s["zero_points"], s["k"], s["group"]).float()
    w = (_codes(s["codes"]).float() - zero) * _spread(s["scales"], s["k"], s["group"])
    y = torch.matmul(s["x"].float(), w.t())
    if s["b"] is not None:
        y = y + s["b"].float()
    return y.to(s["x"].dtype)


def _round(v):
    """Half away from zero (in 64 bits: adding a half would round in 32)."""
    return (torch.sign(v) * torch.floor(v.abs().double() + 0.5)).float()


def _quantize_w4(s):
    w, group = s["w"], s["group"]
    n, k = w.shape
    groups = -(-k // group)
    x = torch.nn.functional.pad(w, (0, groups * group - k)).view(n, groups, group)
    if s["zeros"]:
        lo, hi = x.amin(-1).clamp(max=0.0), x.amax(-1).clamp(min=0.0)
        scale = (hi - lo) / 15.0
        scale = torch.where(scale == 0, 1.0, scale)
        zero = _round(-lo / scale).clamp(0, 15)
        code = (_round(x / scale[..., None]) + zero[..., None]).clamp(0, 15) - zero[..., None]
    else:
        scale = x.abs().amax(-1) / 7.0
        scale = torch.where(scale == 0, 1.0, scale)
        zero = None
        code = _round(x / scale[..., None]).clamp(-8, 7)
    values = (code * scale[..., None]).view(n, -1)[:, :k].contiguous()
    return values, scale, None if zero is None else zero.to(torch.uint8)


# ---- what a pass cannot do without ----------------------------------------------


def work(case):
    c = case
    if c["kind"] == "append":
        tokens = sum(_lens(c)[0])
        each = tokens * c["d"]
        moved = each * (2 * c["h"] + 2 * c["hkv"]) * _BYTES[c["type"]] + each * 2 * c["hkv"] * _BYTES[c["cache"]]
        return {"bytes": moved + tokens * 4 * (c["rot"] + 1), "flops": 3 * tokens * (c["h"] + c["hkv"]) * c["rot"]}
    if c["kind"] == "attention":
        rows = pairs = tokens = 0
        for q, kv in zip(*_lens(c)):
            w = c["window"] or kv
            first = kv - q + 1  # keys that the first new token sees, without a window
            rows += min(kv, q + w - 1)
            full = max(0, min(q, w - first + 1))  # tokens that see fewer keys than the window
            pairs += full * first + full * (full - 1) // 2 + (q - full) * w
            tokens += q
        return {"bytes": 2 * rows * c["hkv"] * c["d"] * _BYTES[c["cache"]]
                + 2 * tokens * c["h"] * c["d"] * _BYTES[c["type"]], "flops": 4 * pairs * c["h"] * c["d"]}
    n, k, groups = c["n"], c["k"], -(-c["k"] // c["group"])
    weight = n * k // 2 + n * groups * (5 if c["zeros"] else 4)
    if c["kind"] == "linear_w4":
        b = _BYTES[c["type"]]
        return {"bytes": weight + b * (c["m"] * (k + n) + (n if c["bias"] else 0)), "flops": 2 * c["m"] * n * k}
    return {"bytes": 8 * n * k + 2 * weight, "flops": 4 * n * k}


# ---- the same results in 64 bits --------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _append64, "attention": _attention64, "linear_w4": _linear64, "quantize_w4": _scales64}[s["kind"]](s)


def _append64(s):
    k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    off, kl = s["q_offsets"].tolist(), s["kv_lens"].tolist()
    r = s["rot"]
    # dims that meet: (first, second) of every pair
    first = torch.arange(0, r, 2, device="cuda") if s["inter"] else torch.arange(r // 2, device="cuda")
    second = first + 1 if s["inter"] else first + r // 2

    def turn(x, at):
        y = x.double()
        z = torch.complex(y[..., first], y[..., second]) * torch.complex(s["cos"][at].double(), s["sin"][at].double())[:, None]
        y[..., first], y[..., second] = z.real, z.imag
        return y

    for n in range(s["seqs"]):
        a, b = off[n], off[n + 1]
        at = torch.arange(kl[n] - (b - a), kl[n], device="cuda")
        out[a:b] = turn(s["q"][a:b], at)
        where = (s["page_table"][n].long()[at // s["page"]], at % s["page"])
        k_pages[where], v_pages[where] = turn(s["k"][a:b], at), s["v"][a:b].double()
    return out, k_pages, v_pages


def _attention64(s):
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    off, kl, g = s["q_offsets"].tolist(), s["kv_lens"].tolist(), s["h"] // s["hkv"]
    for n in range(s["seqs"]):
        a, b, kv = off[n], off[n + 1], kl[n]
        at = s["page_table"][n, :-(-kv // s["page"])].long()
        k = s["k_pages"][at].flatten(0, 1)[:kv].double()
        v = s["v_pages"][at].flatten(0, 1)[:kv].double()
        i = torch.arange(kv - (b - a), kv, device="cuda")[:, None]
        j = torch.arange(kv, device="cuda")[None]
        hidden = (j > i) | (j + s["window"] <= i) if s["window"] else j > i
        for h in range(s["h"]):
            w = s["q"][a:b, h].double() @ k[:, h // g].t() / math.sqrt(s["d"])
            out[a:b, h] = torch.softmax(w.masked_fill(hidden, -math.inf), -1) @ v[:, h // g]
    return out


def _linear64(s):
    byte = s["codes"].long()
    w = torch.empty(s["n"], s["k"], dtype=torch.float64, device="cuda")
    w[:, 0::2], w[:, 1::2] = (byte % 16).double(), (byte // 16).double()
    group = torch.arange(s["k"], device="cuda") // s["group"]
    w -= 8.0 if s["zero_points"] is None else s["zero_points"].double()[:, group]
    w *= s["scales"].double()[:, group]
    y = s["x"].double() @ w.t()
    return y if s["b"] is None else y + s["b"].double()


def _scales64(s):
    # (codes next to a border between two of them go by the scale's last bit in
    # fp32: the scales have a value in 64 bits, the codes have none)
    w = s["w"].double()
    k, group = s["k"], s["group"]
    cut = [w[:, i:i + group] for i in range(0, k, group)]
    if s["zeros"]:
        span = [x.amax(1).clamp(min=0) - x.amin(1).clamp(max=0) for x in cut]
        return None, torch.stack(span, 1) / 15, None
    return None, torch.stack([x.abs().amax(1) for x in cut], 1) / 7, None
