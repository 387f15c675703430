"""Plain forms of values in 4 bits and of rotation, in float64, for the tests of the paged
cache that holds them."""

from __future__ import annotations

import torch

from paged_test_utils import DEV, Cache

# (2^-200 to 2^200: a device's pow may be a rounding off)
POWERS = [2.0 ** n for n in range(-200, 201)]
STEPS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def power(e):
    return torch.tensor(POWERS, dtype=torch.float64, device=e.device)[e.long() + 200]


def held4(x):
    """(values (..., D) float64, scale bytes (..., D / 32)) that 4-bit pages hold of x."""
    b = x.double().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1)
    bad = ~torch.isfinite(b).all(-1)
    e = torch.full_like(top, -125.0)
    # the smallest power of two of which the largest is at most 7, by trying them all
    for n in range(125, -126, -1):
        e = torch.where(top <= 7.0 * 2.0 ** n, float(n), e) if n < 125 else torch.full_like(e, 125.0)
    s = power(e)[..., None]
    a = b.abs() / s
    steps = torch.tensor(STEPS, dtype=torch.float64, device=x.device)
    far = (a[..., None] - steps).abs()
    near = far.amin(-1, keepdim=True)
    # of two that are as near the even one
    even = torch.arange(8, device=x.device) % 2 == 0
    code = torch.where((far == near) & even, 2, (far == near).int()).argmax(-1)
    code = torch.where(a >= 6.0, 7, code)
    v = steps[code] * s * torch.where(b < 0, -1.0, 1.0)
    v = torch.where(bad[..., None], float("nan"), v)
    return v.flatten(-2), torch.where(bad, 255, e.int() + 127)


def parts4(pages):
    """Codes' bytes (P, NKVH, page, D / 2) and scales (P, NKVH, D / 32, page), as views."""
    P, H, ps, row = pages.shape
    D = row // 17 * 32
    codes = pages.as_strided((P, H, ps, D // 2), (*pages.stride()[:2], D // 2, 1),
                             pages.storage_offset())
    return codes, pages.as_strided((P, H, D // 32, ps), (*pages.stride()[:2], ps, 1),
                                   pages.storage_offset() + ps * D // 2)


def values4(pages):
    """Values (P, NKVH, page, D), float64."""
    codes, scales = parts4(pages)
    n = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    v = torch.tensor(STEPS, dtype=torch.float64, device=pages.device)[n & 7]
    v = torch.where(n >= 8, -v, v)
    s = power(scales.long() - 127)
    s = torch.where(scales == 255, float("nan"), s).transpose(2, 3)
    return v * s.repeat_interleave(32, -1)


class Cache4(Cache):
    """``Cache`` with pages of random codes and scales: k_pages, v_pages are the bytes, k and v
    the values (float64).  layout "apart": pages and heads with gaps between them."""

    def __init__(self, lens, NKVH, D, page, seed, layout="dense", **kw):
        super().__init__(lens, NKVH, D, page, torch.float32, seed, **kw)
        row = D // 2 + D // 32

        def pages():
            n = page * row + (0 if layout == "dense" else 48)
            flat = torch.randint(0, 256, (self.P, NKVH, n), generator=self.g, device=DEV,
                                 dtype=torch.uint8)
            x = flat[..., :page * row].unflatten(-1, (page, row))
            s = parts4(x)[1]
            s.copy_(torch.randint(123, 128, s.shape, generator=self.g, device=DEV))
            return x

        self.k_pages, self.v_pages = pages(), pages()
        self.decode()

    def decode(self):
        self.k, self.v = values4(self.k_pages), values4(self.v_pages)


def rotated64(x, cos, sin, pos, eps):
    """x (n, heads, D) at positions pos (n), float64; rows of negative positions are 0."""
    x, at = x.double(), pos.clamp(min=0).long()
    c, s = cos[at].double()[:, None], sin[at].double()[:, None]
    a, b = x.chunk(2, -1)
    y = torch.cat([a * c + b * s, b * c - a * s], -1)
    if eps is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt()
    return torch.where((pos >= 0)[:, None, None], y, 0.0)
