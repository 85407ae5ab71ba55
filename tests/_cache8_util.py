"""Helpers for the tests of the paged cache in 8 bits: its definition in 64 bits."""
import torch

F8 = torch.float8_e4m3fn


def rounded(x):
    """To the nearest code, ties to even (x up to 448 in magnitude), as a 64-bit number."""
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
    step = torch.exp2(e - 3)
    return torch.round(x / step) * step


def values(pages, scales):
    """What a cache stands for, in 64 bits."""
    return pages.float().double() * scales.double()[:, None, :, None]


def write(x, pages, scales, slots):
    """WRITE of keys or of values, a token's page after the other: new (codes as 64-bit numbers, scales)."""
    codes, scales = pages.float().double().cpu(), scales.double().cpu().clone()
    x, page, P = x.double().cpu(), pages.shape[1], pages.shape[0]
    of = {}
    for i, s in enumerate(slots.tolist()):
        if 0 <= s < P * page:
            of.setdefault(s // page, []).append((i, s % page))
    for p, tokens in of.items():
        first = min(r for _, r in tokens)
        new = x[[i for i, _ in tokens]]
        top = torch.where(torch.isfinite(new), new.abs(), torch.zeros_like(new)).amax((0, 2))
        scale = torch.exp2(torch.ceil(torch.log2(top / 448.0)).clamp(min=-100.0))
        if first > 0:
            scale = torch.maximum(scale, scales[p])
            codes[p, :first] = rounded(codes[p, :first] * (scales[p] / scale)[:, None])
        for (i, r), z in zip(tokens, new):
            codes[p, r] = torch.where(torch.isfinite(z), rounded(z / scale[:, None]), torch.full_like(z, float("nan")))
        scales[p] = scale
    return codes, scales
