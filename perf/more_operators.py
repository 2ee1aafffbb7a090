"""Performance cases of a decode step over an 8-bit cache: norms and rotary
positions on the way into the pages, the cache read back, attention over it,
and the choice of the next token.

  append     queries and keys of every head normed and turned, k / v written
             into the pages of a ragged batch: in 8 bits (then the new rows are
             read back as the values that they stand for) or in 16
  read       the cached rows of whole sequences as dense values, as a program
             does that hands a prefix over or saves it
  attention  that batch's new tokens (one each, or chunks of a prompt) over
             8-bit pages: causal, with an optional window, grouped heads
  sample     tokens from logits, and the logarithms of their probabilities:
             temperature, top-k, top-p and min-p of each row, random numbers
             given

An 8-bit row (a position's key or value of one head) is d codes c and a byte b
for its step s = (8 + b % 8) 2^(b // 8 - 22), and stands for (c - 128) s.  b
is the smallest up to 207 with 127 s >= the row's largest magnitude.

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
_BYTES = {"f32": 4, "bf16": 2, "f16": 2, "u8": 1}
_EPS = 1e-6


def _gh():
    pkg = os.path.join(os.getcwd(), "ghost-flow_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import ghostflow_hip
    return ghostflow_hip


def listed():
    return [
        # one decode step of 64 sequences, norms and 8 bits: latency of the step
        {"name": "append_decode_64_q8", "kind": "append", "type": "bf16", "cache": "u8", "h": 32, "hkv": 8, "d": 128,
         "seqs": 64, "q": 1, "kv": 4096, "page": 16, "rot": 128, "inter": False, "norm": True},
        # four long prompts in fp32 into 8 bits
        {"name": "append_prompts_q8", "kind": "append", "type": "f32", "cache": "u8", "h": 32, "hkv": 8, "d": 128,
         "seqs": 4, "q": 4000, "kv": 4000, "page": 64, "rot": 128, "inter": False, "norm": False},
        # prompts with normed heads into a 16-bit cache, half of a head turned
        {"name": "append_prompts_norm_bf16", "kind": "append", "type": "bf16", "cache": "bf16", "h": 16, "hkv": 4,
         "d": 128, "seqs": 8, "q": 2500, "kv": 2600, "page": 32, "rot": 64, "inter": True, "norm": True},
        # a short prefix of one user handed over: latency
        {"name": "read_1_f16", "kind": "read", "type": "f16", "cache": "u8", "h": 12, "hkv": 12, "d": 64, "seqs": 1,
         "q": 517, "kv": 517, "page": 16},
        # the caches of 16 sequences in fp32
        {"name": "read_16_f32", "kind": "read", "type": "f32", "cache": "u8", "h": 32, "hkv": 8, "d": 128, "seqs": 16,
         "q": 4096, "kv": 4096, "page": 16},
        # a single user's next token, small heads: latency
        {"name": "attn_decode_1_f16", "kind": "attention", "type": "f16", "cache": "u8", "h": 12, "hkv": 12, "d": 64,
         "seqs": 1, "q": 1, "kv": 517, "page": 16, "window": 0},
        # the decode step of a loaded server
        {"name": "attn_decode_64_bf16", "kind": "attention", "type": "bf16", "cache": "u8", "h": 32, "hkv": 8, "d": 128,
         "seqs": 64, "q": 1, "kv": 4096, "page": 16, "window": 0},
        # chunks of several prompts beside sequences that decode, the
        # framework's own fp32 over 8 bits, with a window
        {"name": "attn_mixed_f32", "kind": "attention", "type": "f32", "cache": "u8", "h": 32, "hkv": 8, "d": 128,
         "seqs": 6, "q": 700, "kv": 3000, "page": 16, "window": 1024},
        # a chunk of a long prompt
        {"name": "attn_chunk_2048_bf16", "kind": "attention", "type": "bf16", "cache": "u8", "h": 32, "hkv": 8,
         "d": 128, "seqs": 1, "q": 2048, "kv": 16384, "page": 64, "window": 0},
        # one user's next token: latency
        {"name": "sample_1_f32", "kind": "sample", "type": "f32", "rows": 1, "vocab": 32000, "filters": "both"},
        # a loaded server's tokens, every row with its own settings
        {"name": "sample_64_bf16", "kind": "sample", "type": "bf16", "rows": 64, "vocab": 131072, "filters": "mixed"},
        # many rows drawn from all of an odd vocabulary
        {"name": "sample_256_f32", "kind": "sample", "type": "f32", "rows": 256, "vocab": 50257, "filters": "none"},
    ]


# ---- drawing more cases of the same ranges ------------------------------------


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    return rng.choice(((32, 8, 128), (32, 32, 128), (12, 12, 64), (16, 4, 64), (8, 1, 128), (28, 4, 128), (20, 5, 80),
                       (16, 2, 96)))


def draw(rng):
    while True:
        c = _draw(rng)
        if c["kind"] == "attention" and 4 * c["seqs"] * c["h"] * c["q"] * c["kv"] > 5e9:
            continue  # scores of the plain form
        if "kv" in c and c["seqs"] * c["kv"] * c["hkv"] * c["d"] > 3e8:
            continue  # pages
        if c["kind"] == "sample" and c["rows"] * c["vocab"] > 1.5e7:
            continue
        w = work(c)
        if w["flops"] <= 5e11 and w["bytes"] <= 6e8:
            return c


def _draw(rng):
    kind = rng.choice(("append", "append", "read", "attention", "attention", "attention", "sample", "sample"))
    if kind == "sample":
        return {"kind": kind, "type": rng.choice(("f32", "bf16", "f16")), "rows": _log(rng, 1, 256),
                "vocab": _log(rng, 1000, 131072), "filters": rng.choice(("both", "mixed", "mixed", "none"))}
    (h, hkv, d), t = _heads(rng), rng.choice(("bf16", "bf16", "f16", "f32"))
    seqs = _log(rng, 1, 64)
    q = 1 if kind != "read" and rng.random() < 0.5 else _log(rng, 2, 2048 if kind == "attention" else 4000)
    c = {"kind": kind, "type": t, "cache": "u8", "h": h, "hkv": hkv, "d": d, "seqs": seqs, "q": q,
         "kv": q if kind == "read" else max(q, _log(rng, 64, 16384)), "page": rng.choice((16, 16, 32, 64, 100, 128))}
    if kind == "append":
        c.update(rot=rng.choice((d, d, d // 2)), inter=rng.random() < 0.3, norm=rng.random() < 0.7)
        if c["norm"] and rng.random() < 0.25:
            c["cache"] = t
    elif kind == "attention":
        c.update(window=0 if rng.random() < 0.6 else _log(rng, 100, 4096))
    return c


# ---- what a program has in hand -------------------------------------------------


def _lens(c):
    """New tokens and positions of every sequence: the first has the most, the
    others between a quarter and all of it, every third of a batch of chunks a
    single token.  What is read back are whole sequences."""
    r = random.Random(c["seqs"] * 1000003 + c["kv"] * 1009 + c["q"])
    ql, kl = [], []
    for s in range(c["seqs"]):
        q = c["q"] if s == 0 else 1 if s % 3 == 2 else r.randint(max(1, c["q"] // 4), c["q"])
        kv = c["kv"] if s == 0 else r.randint(max(1, c["kv"] // 4), c["kv"])
        ql.append(kv if c["kind"] == "read" else q)
        kl.append(max(ql[-1], kv))
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
    n = order.numel()
    shape = (n, c["page"], c["hkv"], c["d"])
    # (whole pages hold something: what earlier sequences left there)
    if c["cache"] != "u8":
        s["k_pages"] = torch.randn(shape, generator=g, device="cuda").to(_TYPES[c["cache"]])
        s["v_pages"] = torch.randn(shape, generator=g, device="cuda").to(_TYPES[c["cache"]])
        s["k_scales"] = s["v_scales"] = None
        return
    for x in ("k", "v"):
        # normal values whose rows have a largest magnitude of 2.4 to 3.5
        code = torch.randn(shape, generator=g, device="cuda").mul_(43.0).round_().clamp_(-127, 127)
        s[x + "_pages"] = code.add_(128).to(torch.uint8)
        s[x + "_scales"] = torch.randint(104, 110, (n, c["hkv"], c["page"]), dtype=torch.uint8, generator=g, device="cuda")
    # the step of every byte
    s["steps"] = torch.tensor([(8 + b % 8) * 2.0 ** (b // 8 - 22) for b in range(208)], device="cuda")


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))

    def normal(*shape, t="f32", std=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * std).to(_TYPES[t])

    s = dict(c)
    if c["kind"] == "sample":
        rows = c["rows"]
        x = normal(rows, c["vocab"], std=2.0)
        # some tens of entries stand out
        x += 9.0 * (torch.rand(x.shape, generator=g, device="cuda") < 40.0 / c["vocab"])
        s["logits"] = x.to(_TYPES[c["type"]])
        s["u"] = torch.rand(rows, generator=g, device="cuda")
        i = torch.arange(rows, device="cuda")
        on, all_rows = torch.ones(rows, device="cuda"), c["filters"] == "both"
        s["temperature"] = 0.6 + 0.7 * torch.rand(rows, generator=g, device="cuda")
        s["top_k"] = torch.zeros(rows, dtype=torch.int32, device="cuda")
        s["top_p"], s["min_p"] = on.clone(), 0 * on
        if c["filters"] != "none":
            # of rows with settings of their own: top-k and top-p, top-p, none,
            # min-p, the likeliest
            k = all_rows | (i % 5 == 0)
            p = all_rows | (i % 5 <= 1)
            s["top_k"][k] = torch.randint(2, 200, (rows,), dtype=torch.int32, generator=g, device="cuda")[k]
            s["top_p"][p] = (0.5 + 0.49 * torch.rand(rows, generator=g, device="cuda"))[p]
            if not all_rows:
                s["min_p"][i % 5 == 3] = 0.05
                s["temperature"][i % 5 == 4] = 0.0
        return s
    _batch(c, g, s)
    if c["kind"] in ("append", "attention"):
        s["q"] = normal(s["tokens"], c["h"], c["d"], t=c["type"])
        s["out"] = torch.zeros_like(s["q"])
    if c["kind"] == "append":
        s["k"] = normal(s["tokens"], c["hkv"], c["d"], t=c["type"], std=1.5)
        s["v"] = normal(s["tokens"], c["hkv"], c["d"], t=c["type"])
        rows = s["page_table"].shape[1] * c["page"]
        freq = 10000.0 ** (-torch.arange(0, c["rot"], 2, dtype=torch.float64, device="cuda") / c["rot"])
        angle = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * freq
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["q_norm"] = 1.0 + normal(c["d"], std=0.2) if c["norm"] else None
        s["k_norm"] = 1.0 + normal(c["d"], std=0.2) if c["norm"] else None
    if c["kind"] == "read" or c["cache"] == "u8" and c["kind"] == "append":
        s["k_out"] = torch.zeros(s["tokens"], c["hkv"], c["d"], dtype=_TYPES[c["type"]], device="cuda")
        s["v_out"] = torch.zeros_like(s["k_out"])
    return s


# ---- one pass -------------------------------------------------------------------


def run(state):
    s = state
    if not own:
        return {"append": _append, "read": _read, "attention": _attention, "sample": _sample}[s["kind"]](s)
    gh = _gh()
    if s["kind"] == "sample":
        return gh.sample(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                         min_p=s["min_p"], want_logprobs=True)
    cache = (s["k_pages"], s["v_pages"], s["page_table"], s["q_offsets"], s["kv_lens"])
    steps = {"k_scales": s["k_scales"], "v_scales": s["v_scales"]}
    if s["kind"] == "attention":
        return gh.paged_attention(s["q"], *cache, causal=True, window=s["window"], max_kv_len=s["max_kv"], out=s["out"],
                                  **steps)
    if s["kind"] == "append":
        gh.paged_append(*cache, s["k"], s["v"], q=s["q"], q_out=s["out"], cos=s["cos"], sin=s["sin"],
                        interleaved=s["inter"], q_norm=s["q_norm"], k_norm=s["k_norm"], norm_eps=_EPS, **steps)
        if s["k_scales"] is None:
            return s["out"], s["k_pages"], s["v_pages"]
    gh.paged_read(*cache, k_out=s["k_out"], v_out=s["v_out"], **steps)
    return (s["out"], s["k_out"], s["v_out"]) if s["kind"] == "append" else (s["k_out"], s["v_out"])


def _rows_of(s):
    """Page, row of it and position of every new token."""
    t = torch.arange(s["tokens"], device="cuda")
    off = s["q_offsets"].long()
    seq = torch.bucketize(t, off[1:], right=True)
    pos = s["kv_lens"].long()[seq] - off[seq + 1] + t
    return s["page_table"][seq, pos // s["page"]].long(), pos % s["page"], pos


def _normed(x, w):
    x = x.float()
    if w is None:
        return x
    # (the sum in 64 bits: 8-bit codes are next to a border now and then)
    r = 1.0 / (x.double().square().mean(-1, keepdim=True) + _EPS).sqrt()
    return x * r.float() * w


def _rotate(x, c, s, rot, inter):
    c, s = c[:, None], s[:, None]
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if inter else (x[..., :rot // 2], x[..., rot // 2:rot])
    p, q = a * c - b * s, b * c + a * s
    y = torch.stack((p, q), -1).flatten(-2) if inter else torch.cat((p, q), -1)
    return torch.cat((y, x[..., rot:]), -1)


def _to_codes(x, steps):
    """Codes and step bytes of rows x [..., d]; halves go away from zero."""
    b = torch.searchsorted(127.0 * steps, x.abs().amax(-1)).clamp(max=207)
    y = x / steps[b][..., None]
    y = torch.sign(y) * torch.floor(y.abs().double() + 0.5).float()
    return (y.clamp(-127, 127) + 128).to(torch.uint8), b.to(torch.uint8)


def _append(s):
    page, row, pos = _rows_of(s)
    c, sn = s["cos"][pos], s["sin"][pos]
    s["out"].copy_(_rotate(_normed(s["q"], s["q_norm"]), c, sn, s["rot"], s["inter"]))
    k, v = _rotate(_normed(s["k"], s["k_norm"]), c, sn, s["rot"], s["inter"]), s["v"].float()
    if s["cache"] != "u8":
        s["k_pages"][page, row] = k.to(s["k_pages"].dtype)
        s["v_pages"][page, row] = v.to(s["v_pages"].dtype)
        return s["out"], s["k_pages"], s["v_pages"]
    for n, x in (("k", k), ("v", v)):
        code, step = _to_codes(x, s["steps"])
        s[n + "_pages"][page, row] = code
        s[n + "_scales"][page, :, row] = step
    return (s["out"],) + _read(s)


def _values(s, n, page, row):
    """Keys or values at pages and rows in fp32."""
    return (s[n + "_pages"][page, row].float() - 128.0) * s["steps"][s[n + "_scales"][page, :, row].long()][..., None]


def _read(s):
    page, row, _ = _rows_of(s)
    for n in ("k", "v"):
        s[n + "_out"].copy_(_values(s, n, page, row))
    return s["k_out"], s["v_out"]


def _attention(s):
    # every sequence padded to the longest
    nq, nk, h, hkv, d = s["max_q"], s["max_kv"], s["h"], s["hkv"], s["d"]
    j = torch.arange(nk, device="cuda")
    page, row = s["page_table"][:, j // s["page"]].long(), (j % s["page"]).expand(s["seqs"], nk)
    k = _values(s, "k", page, row).permute(0, 2, 3, 1).contiguous()  # [S, hkv, d, nk]
    v = _values(s, "v", page, row).transpose(1, 2).contiguous()      # [S, hkv, nk, d]
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


def _sample(s):
    # the largest first, equal ones by their index; sums in 64 bits, for a
    # random number may lie next to a border
    x, at = torch.sort(s["logits"].float(), dim=-1, descending=True, stable=True)
    x = x.double()
    t = s["temperature"].double()[:, None]
    w = torch.exp((x - x[:, :1]) / torch.where(t > 0, t, 1.0))
    n = x.shape[1]
    k = torch.where(s["top_k"] > 0, s["top_k"].long(), n).clamp(max=n)
    k = torch.where(s["temperature"] > 0, k, 1)[:, None]
    i = torch.arange(n, device="cuda")
    w = torch.where(i < k, w, 0.0)
    top_p = s["top_p"].double()[:, None]
    before = torch.cumsum(w, -1) - w
    keep = (i < k) & ((before < top_p * w.sum(-1, keepdim=True)) | (top_p >= 1) | (i == 0))
    keep = keep & ((w >= s["min_p"].double()[:, None]) | (i == 0))
    w = torch.zeros_like(w).scatter_(-1, at, torch.where(keep, w, 0.0))  # by index again
    total = torch.cumsum(w, -1)
    token = (total > s["u"].double()[:, None] * total[:, -1:]).int().argmax(-1, keepdim=True)
    logprob = torch.log(w.gather(-1, token) / total[:, -1:])
    return token[:, 0].to(torch.int32), logprob[:, 0].float()


# ---- what a pass cannot do without ----------------------------------------------


def work(case):
    c = case
    if c["kind"] == "sample":
        n = c["rows"] * c["vocab"]
        # a difference, a product and an exponential of some ten operations
        return {"bytes": n * _BYTES[c["type"]] + c["rows"] * 28, "flops": 12 * n}
    if c["kind"] in ("append", "read"):
        tokens = sum(_lens(c)[0])
        row = 2 * c["hkv"] * (c["d"] * _BYTES[c["cache"]] + (c["cache"] == "u8"))  # of the cache
        dense = 2 * c["hkv"] * c["d"] * _BYTES[c["type"]]
        if c["kind"] == "read":
            return {"bytes": tokens * (row + dense), "flops": 4 * tokens * c["hkv"] * c["d"]}
        qk = (c["h"] + c["hkv"]) * c["d"]
        moved = 2 * c["h"] * c["d"] * _BYTES[c["type"]] + dense + row + 4 * c["rot"]
        flops = 3 * (c["h"] + c["hkv"]) * c["rot"] + 4 * qk * c["norm"]
        if c["cache"] == "u8":  # and read back
            moved += row + dense
            flops += 8 * c["hkv"] * c["d"]
        return {"bytes": tokens * moved, "flops": tokens * flops}
    rows = pairs = tokens = 0
    for q, kv in zip(*_lens(c)):
        w = c["window"] or kv
        first = kv - q + 1  # keys that the first new token sees, without a window
        rows += min(kv, q + w - 1)
        full = max(0, min(q, w - first + 1))  # tokens that see fewer keys than the window
        pairs += full * first + full * (full - 1) // 2 + (q - full) * w
        tokens += q
    return {"bytes": 2 * rows * c["hkv"] * (c["d"] + 1) + 2 * tokens * c["h"] * c["d"] * _BYTES[c["type"]],
            "flops": 4 * pairs * c["h"] * c["d"]}


# ---- the same results in 64 bits --------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _append64, "read": _read64, "attention": _attention64, "sample": _sample64}[s["kind"]](s)


def _positions(s):
    """(first row, its end, positions) of every sequence's new tokens."""
    off, kl = s["q_offsets"].tolist(), s["kv_lens"].tolist()
    return [(a, b, torch.arange(n - (b - a), n, device="cuda")) for a, b, n in zip(off, off[1:], kl)]


def _append64(s):
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    plain = s["cache"] != "u8"
    k_pages, v_pages = (s["k_pages"].double(), s["v_pages"].double()) if plain else (None, None)
    r = s["rot"]
    # dims that meet: (first, second) of every pair
    first = torch.arange(0, r, 2, device="cuda") if s["inter"] else torch.arange(r // 2, device="cuda")
    second = first + 1 if s["inter"] else first + r // 2

    def turn(x, w, at):
        y = x.double()
        if w is not None:
            y = y * w.double() / torch.sqrt(torch.sum(y * y, -1, keepdim=True) / y.shape[-1] + _EPS)
        z = torch.complex(y[..., first], y[..., second]) * torch.complex(s["cos"][at].double(), s["sin"][at].double())[:, None]
        y[..., first], y[..., second] = z.real, z.imag
        return y

    for n, (a, b, at) in enumerate(_positions(s)):
        out[a:b] = turn(s["q"][a:b], s["q_norm"], at)
        if plain:
            where = (s["page_table"][n].long()[at // s["page"]], at % s["page"])
            k_pages[where], v_pages[where] = turn(s["k"][a:b], s["k_norm"], at), s["v"][a:b].double()
    # (8-bit codes and steps next to a border between two of them go by the last
    # bits in fp32: the values they stand for have no value in 64 bits)
    return out, k_pages, v_pages


def _cached64(s, n, x):
    """Sequence n's keys or values."""
    kv = int(s["kv_lens"][n])
    at = s["page_table"][n, :-(-kv // s["page"])].long()
    b = s[x + "_scales"][at].transpose(1, 2).flatten(0, 1)[:kv].long()
    step = torch.ldexp(8.0 + (b % 8).double(), b // 8 - 22)
    return (s[x + "_pages"][at].flatten(0, 1)[:kv].double() - 128) * step[..., None]


def _read64(s):
    return tuple(torch.cat([_cached64(s, n, x) for n in range(s["seqs"])]) for x in ("k", "v"))


def _attention64(s):
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    g = s["h"] // s["hkv"]
    for n, (a, b, i) in enumerate(_positions(s)):
        k, v = _cached64(s, n, "k"), _cached64(s, n, "v")
        j = torch.arange(len(k), device="cuda")[None]
        i = i[:, None]
        hidden = (j > i) | (j + s["window"] <= i) if s["window"] else j > i
        for h in range(s["h"]):
            w = s["q"][a:b, h].double() @ k[:, h // g].t() / math.sqrt(s["d"])
            out[a:b, h] = torch.softmax(w.masked_fill(hidden, -math.inf), -1) @ v[:, h // g]
    return out


def _sample64(s):
    out = torch.empty(s["rows"], dtype=torch.int32, device="cuda")
    logprob = torch.zeros(s["rows"], dtype=torch.float64, device="cuda")
    for r in range(s["rows"]):
        x = s["logits"][r].double()
        t, k, p, least, u = (float(s[n][r]) for n in ("temperature", "top_k", "top_p", "min_p", "u"))
        # (the first of the largest)
        best = int(torch.nonzero(x == x.max())[0])
        if t <= 0:
            out[r] = best
            continue
        rank = torch.argsort(x, descending=True, stable=True)
        if k > 0:
            rank = rank[:int(k)]
        prob = torch.softmax(x[rank] / t, 0)
        if p < 1:
            ahead = torch.cat((prob.new_zeros(1), prob.cumsum(0)[:-1]))
            stay = max(1, int((ahead < p).sum()))
            rank, prob = rank[:stay], prob[:stay]
        stay = prob >= least * prob[0]
        rank = rank[stay].sort().values
        prob = torch.softmax(x[rank] / t, 0)
        n = min(int((prob.cumsum(0) <= u).sum()), len(rank) - 1)
        out[r], logprob[r] = rank[n], prob[n].log()
    return out, logprob
