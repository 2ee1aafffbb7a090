"""4-bit weights in groups for the tests: the formulas in plain torch (CPU)."""
import torch

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def spread(v, k, group):
    return v.repeat_interleave(group, 1)[:, :k]


def unpack(codes):
    return torch.stack((codes & 15, codes >> 4), -1).flatten(1)


def weight(codes, scales, zps, group):
    """W' in 64 bits."""
    k = codes.shape[1] * 2
    z = 8.0 if zps is None else spread(zps, k, group).double()
    return (unpack(codes).double() - z) * spread(scales, k, group).double()


def rounded(v):
    """Half away from zero of fp32 values."""
    return (torch.sign(v) * torch.floor(v.abs().double() + 0.5)).float()


def quantize(w, group, symmetric):
    """(codes, scales, zero points) with the scheme's fp32 arithmetic."""
    n, k = w.shape
    groups = -(-k // group)
    x = torch.nn.functional.pad(w, (0, groups * group - k)).view(n, groups, group)
    if symmetric:
        s = x.abs().amax(-1) * torch.tensor(1 / 7, dtype=torch.float32)
        s = torch.where(s == 0, torch.ones(()), s)
        z = None
        c = rounded(x / s[..., None]).clamp(-8, 7) + 8
    else:
        lo, hi = x.amin(-1).clamp(max=0.0), x.amax(-1).clamp(min=0.0)
        s = (hi - lo) * torch.tensor(1 / 15, dtype=torch.float32)
        s = torch.where(s == 0, torch.ones(()), s)
        z = rounded(-lo / s).clamp(0, 15)
        c = (rounded(x / s[..., None]) + z[..., None]).clamp(0, 15)
    c = c.reshape(n, -1)[:, :k].to(torch.uint8)
    return c[:, 0::2] | c[:, 1::2] << 4, s, None if z is None else z.to(torch.uint8)


def random_weight(n, k, group, zeros, seed, exact=False):
    g = torch.Generator().manual_seed(seed)
    groups = -(-k // group)
    codes = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, generator=g)
    if exact:  # powers of two
        scales = 2.0 ** torch.randint(-2, 2, (n, groups), generator=g).float()
    else:
        scales = torch.rand(n, groups, generator=g) * 0.02 + 1e-3
    zps = torch.randint(0, 16, (n, groups), dtype=torch.uint8, generator=g) if zeros else None
    return codes, scales, zps
