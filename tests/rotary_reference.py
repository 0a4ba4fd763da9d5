"""64-bit definitions of the rotary operators and the error bounds that their tests use (see ``training_reference``)."""

from __future__ import annotations

import math
from fractions import Fraction

import torch

from training_reference import U, acc, floor, half

# An angle is reduced to a fraction of a turn, rounded to fp32 (at most 1/2, so pi U of the angle), and its sine and
# cosine are off by at most 2 U of themselves and U for the factor: 6.2 U. Two products and a sum add 2 U to each term.
TURN = 10 * U
# For 16-bit tensors the functions are off by 2^-21.19 (7 U) in place of 2 U of themselves, and their argument rounds once
# more (2 pi t: pi U) and carries 2 pi's own rounding (U / 2 of half a turn, 2 U): 10.2 U more.
TURN16 = 21 * U


def turn_error(t: torch.dtype) -> float:
    return TURN if t == torch.float32 else TURN16


# A head's sum of squares has at most 13 roundings in a row and one in each square, the mean two, eps one, the reciprocal
# root 4 U, and the root halves what is before it: 13 U. x r gamma: two more.
RSTD = 13 * U
# 2 pi to 80 digits: A000796 doubled.
PI = Fraction(31415926535897932384626433832795028841971693993751058209749445923078164062862090, 10**79)


def exact_angle(position: int, freq: float) -> float:
    """position * freq modulo 2 pi, by rational arithmetic."""
    a = Fraction(position) * Fraction(freq)
    return float(a - round(a / (2 * PI)) * 2 * PI)


def angles(q, freqs, positions):
    """[..., length, 1, pairs] in 64 bits; positions below 2^24, so that the product loses nothing that counts."""
    p = torch.arange(q.shape[-3], device=q.device) if positions is None else positions
    return (p.double()[..., None] * freqs.double())[..., None, :]


def turned(x, angle, interleaved, scale):
    n = angle.shape[-1]
    c, s = angle.cos() * scale, angle.sin() * scale
    if interleaved:
        a, b = x[..., :2 * n:2], x[..., 1:2 * n:2]
        y = torch.stack((a * c - b * s, a * s + b * c), -1).flatten(-2)
    else:
        a, b = x[..., :n], x[..., n:2 * n]
        y = torch.cat((a * c - b * s, a * s + b * c), -1)
    return torch.cat((y, x[..., 2 * n:]), -1)


def pair_size(x, n, interleaved, scale):
    """|a| + |b| of each dim's pair times the factor, 0 behind the pairs."""
    x = x.abs()
    rest = torch.zeros_like(x[..., 2 * n:])
    if interleaved:
        s = (x[..., :2 * n:2] + x[..., 1:2 * n:2]).repeat_interleave(2, -1)
    else:
        s = (x[..., :n] + x[..., n:2 * n]).repeat(*[1] * (x.dim() - 1), 2)
    return torch.cat((s * abs(scale), rest), -1)


def rotary_reference(x, freqs, positions, interleaved, scale, inverse):
    """(value, bound)."""
    t, n = x.dtype, freqs.shape[0]
    x = x.double()
    a = angles(x, freqs, positions)
    y = turned(x, -a if inverse else a, interleaved, scale)
    return y, half(t) * y.abs() + turn_error(t) * pair_size(x, n, interleaved, scale) + floor(t) + 2.0**-149


def qk_norm_reference(x, dy, gamma, freqs, positions, interleaved, scale, eps, lens):
    """{"y", "dx", "dgamma": (value, bound)} of one side; gradients by the formula."""
    t = x.dtype
    hd = x.shape[-1]
    tw = torch.float32 if gamma is None else gamma.dtype
    f = torch.zeros(0, device=x.device, dtype=torch.float64) if freqs is None else freqs
    g = torch.ones(hd, device=x.device, dtype=torch.float64) if gamma is None else gamma.double()
    x, dy = x.double(), dy.double()
    inside = torch.ones(x.shape[:-2], dtype=torch.bool, device=x.device)
    if lens is not None:
        row = torch.arange(x.shape[-3], device=x.device)
        inside = (row < lens.view(-1, 1)).view(x.shape[:-2])
    inside = inside[..., None, None]
    x, dy = torch.where(inside, x, 0.0), torch.where(inside, dy, 0.0)
    a = angles(x, f, positions)
    r = ((x * x).mean(-1, keepdim=True) + eps) ** -0.5
    r = torch.where(inside, r, 0.0)
    xhat = x * r
    z = xhat * g
    y = turned(z, a, interleaved, scale)
    n = f.shape[0]
    e_z = (RSTD + 2 * U) * z.abs()
    small = 2.0**-149
    e_y = half(t) * y.abs() + turn_error(t) * pair_size(z, n, interleaved, scale) + turn_bound(e_z, n, interleaved, scale) + \
        floor(t) + small
    gr = turned(dy, -a, interleaved, scale)
    e_g = turn_error(t) * pair_size(dy, n, interleaved, scale)
    h = gr * g
    e_h = e_g * g.abs() + U * h.abs()
    m = (h * xhat).mean(-1, keepdim=True)
    size = (h * xhat).abs().mean(-1, keepdim=True)
    # 13 roundings of the sum and one of each product, r, and the mean's two.
    e_m = (e_h * xhat.abs()).mean(-1, keepdim=True) + (16 * U + RSTD) * size
    dx = r * (h - xhat * m)
    e_dx = half(t) * dx.abs() + r * (e_h + xhat.abs() * e_m) + \
        (2 * RSTD + 6 * U) * r * (h.abs() + xhat.abs() * m.abs()) + floor(t) + small
    rows = x[..., 0].numel()
    terms = gr * xhat
    dg = terms.flatten(0, -2).sum(0)
    e_dg = half(tw) * dg.abs() + (acc(rows) * terms.abs() + e_g * xhat.abs() + (RSTD + 2 * U) * terms.abs()
                                  ).flatten(0, -2).sum(0) + floor(tw) + small
    return {"y": (y, e_y), "dx": (dx, e_dx), "dgamma": (dg, e_dg)}


def turn_bound(e, n, interleaved, scale):
    """What an error e of the dims becomes at most by the rotation."""
    return torch.cat((pair_size(e, n, interleaved, scale)[..., :2 * n], e[..., 2 * n:]), -1)


def check_pi() -> bool:
    return abs(float(PI) - math.pi) < 1e-15
