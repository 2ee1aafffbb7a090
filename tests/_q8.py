"""A paged cache of 8 bits for the tests: the rule of codes and steps in plain
torch on the CPU, and batches over such a cache."""
import torch

import _paged as P

STEPS = torch.tensor([(8 + b % 8) * 2.0 ** (b // 8 - 22) for b in range(208)])
LARGEST = 127 * 120.0


def quantise(x):
    """(codes, step bytes) of rows x [..., d] in fp32."""
    x = torch.nan_to_num(x.float(), nan=0.0, posinf=float("inf"), neginf=float("-inf"))
    b = torch.searchsorted(127.0 * STEPS, x.abs().amax(-1).contiguous()).clamp(max=207)
    y = x / STEPS[b][..., None]
    y = torch.where(y.isinf(), y, torch.sign(y) * torch.floor(y.abs().double() + 0.5).float())
    return (y.clamp(-127, 127) + 128).to(torch.uint8), b.to(torch.uint8)


def values(codes, steps):
    return (codes.float() - 128) * STEPS[steps.long().clamp(max=207)][..., None]


def normed(x, w, eps):
    x = x.float()
    if w is None:
        return x
    r = 1.0 / (x.double().square().mean(-1, keepdim=True) + eps).sqrt()
    return x * r.float() * w


def turned(x, pos, cos, sin, interleaved):
    """x [heads, d] at a position, every fp32 operation rounded by itself."""
    y = x.float().clone()
    if cos is None:
        return y
    i = torch.arange(cos.shape[1])
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + cos.shape[1])
    c, s = cos[pos], sin[pos]
    y[:, a], y[:, b] = x[:, a] * c - x[:, b] * s, x[:, b] * c + x[:, a] * s
    return y


def batch(q_lens, kv_lens, *, kind="bf16", size=1.0, steps_like="rows", **kw):
    """_paged.batch with its pages in 8 bits: codes, and step bytes in
    k_scales / v_scales [pages, kv_heads, page].  Rows without a position hold any
    codes and bytes (255 among them).  steps_like "pages": bytes of a page's
    heads lie 3 bytes apart from one another."""
    b = P.batch(q_lens, kv_lens, types=(kind, "f32"), **kw)
    g = torch.Generator().manual_seed(7)
    for x in ("k", "v"):
        pages = b[x + "_pages"]
        n, page, heads, d = pages.shape
        codes, steps = quantise(pages * size)
        stale = pages.isnan().all(-1)
        codes[stale] = torch.randint(0, 256, (int(stale.sum()), d), dtype=torch.uint8, generator=g)
        steps[stale] = torch.tensor([255, 208, 3, 207], dtype=torch.uint8)[torch.arange(int(stale.sum())) % 4]
        if pages.stride(1) < pages.stride(2):  # the heads' rows together
            b[x + "_pages"] = codes.transpose(1, 2).contiguous().transpose(1, 2)
        else:
            b[x + "_pages"] = codes.contiguous()
        wide = torch.zeros(n, heads, page + (3 if steps_like == "pages" else 0), dtype=torch.uint8)
        wide[..., :page] = steps.transpose(1, 2)
        b[x + "_scales"] = wide[..., :page]
    return b


def plain(b):
    """The same batch over the values that the cache holds."""
    out = dict(b)
    for x in ("k", "v"):
        out[x + "_pages"] = values(b[x + "_pages"], b[x + "_scales"].transpose(1, 2))
    return out


def to(b, dev):
    out = {}
    for n, t in b.items():
        if not torch.is_tensor(t):
            out[n] = t
        elif n.endswith("_scales"):
            base = t._base if t._base is not None else t
            out[n] = base.to(dev)[..., :t.shape[-1]]
        elif n.endswith("_pages") and not t.is_contiguous():
            out[n] = t.transpose(1, 2).to(dev).transpose(1, 2)
        else:
            out[n] = t.to(dev)
    return out


def scales(b):
    return {"k_scales": b["k_scales"], "v_scales": b["v_scales"]}
