"""The AdamW update in 64 bits with its bounds, and the 8-bit moments from their description (see ``training_reference``)."""

from __future__ import annotations

import torch

from training_reference import U, floor, half

# Magnitudes of the codes relative to their block's largest: 1 is the top code, each octave below has 8 (m) or 16 (u) steps.
M_TABLE = torch.tensor([0.0] + [(1 + (c % 8) / 8) * 2.0 ** (c // 8) for c in range(1 - 127, 1)], dtype=torch.float64)
U_TABLE = torch.tensor([0.0] + [(1 + (c % 16) / 16) * 2.0 ** (c // 16) for c in range(1 - 255, 1)], dtype=torch.float64)


def values(codes: torch.Tensor, top: torch.Tensor, table: torch.Tensor) -> torch.Tensor:
    """fp32 products of the codes' magnitudes (exact in fp32) and their blocks' scales."""
    c = codes.long()
    rel = table.to(c.device)[c & 127 if len(table) == 128 else c].float()
    v = (rel.view(-1, 256) * top[:, None]).view(-1)
    return torch.where(codes >= 128, -v, v) if len(table) == 128 else v


def codes(x: torch.Tensor, table: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales) of finite fp32 values: the nearest table entry, ties to the even mantissa, by search."""
    top = x.view(-1, 256).abs().amax(1)
    inv = torch.where(top >= torch.finfo(torch.float32).tiny, 1 / top, 0.0)
    r = (x.abs().view(-1, 256) * inv[:, None]).view(-1).double()
    t = table.to(x.device)
    mid = (t[1:] + t[:-1]) / 2  # exact in 64 bits
    lo = torch.bucketize(r, mid)  # entries with mid < r lie below
    tie = (lo < len(mid)) & (r == mid[lo.clamp(max=len(mid) - 1)])
    lo = torch.where(tie & (lo > 0) & (lo % 2 == 0), lo + 1, lo)  # odd codes have even mantissas
    if len(t) == 128:
        return torch.where(x < 0, lo + 128, lo).to(torch.uint8), top
    return torch.where((lo == 0) & (r > 0), 1, lo).to(torch.uint8), top


def adamw_reference(p, g, m, v, t, lr, betas, eps, wd, gs):
    """{"p", "m", "v": (value, bound)} of one tensor, from the moments' values; and m, u in fp32 as the codes are made."""
    (b1, b2), typ = betas, p.dtype
    f = torch.tensor(gs, dtype=torch.float32, device=p.device)
    g32 = g.float() * f
    m32 = m * b1 + g32 * (1 - b1)
    v32 = v * b2 + (g32 * g32) * (1 - b2)
    p, g, m, v = p.double(), g.double() * f.double(), m.double(), v.double()
    m_new, v_new = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    tiny = 2.0**-149
    # Factors and products round once each, the sum once; the gradient's factor once (twice in its square).
    e_m = 5 * U * (b1 * m.abs() + (1 - b1) * g.abs()) + 4 * tiny
    e_v = 7 * U * v_new + 4 * tiny
    size, root = lr / (1 - b1**t), (1 - b2**t) ** -0.5
    u = v_new.sqrt()
    denom = u * root + eps
    step = size * m_new / denom
    # Root: half of its argument's error, one of its own; factor, product, sum, quotient, size, product: 12 U.
    e_step = size * e_m / denom + 12 * U * step.abs() + torch.where(v_new < 1e-36, step.abs(), 0.0)
    new = (1 - lr * wd) * p - step
    e_p = half(typ) * new.abs() + e_step + 4 * U * (p.abs() + step.abs()) + floor(typ) + tiny
    return {"p": (new, e_p), "m": (m_new, e_m), "v": (v_new, e_v)}, m32, v32.sqrt()
