"""64-bit definitions of the training operators and the error bounds that their tests use.

Bounds count roundings. ``half(t)`` is half a step of type t relative to the value (bf16 2^-8, fp16 2^-11, fp32 2^-24):
what one rounding may cost. A sum of n fp32 terms is off by at most about n 2^-24 of the sum of their magnitudes;
``acc(n)`` allows four times that, because the tensor cores cut where the FMA pipes round and align products first.
"""

from __future__ import annotations

import math

import torch

U = 2.0**-24


def half(t: torch.dtype) -> float:
    return torch.finfo(t).eps / 2


def floor(t: torch.dtype) -> float:
    """Half of the smallest step of type t: what one rounding costs below its normal range (fp16: under 2^-14)."""
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def acc(n: int) -> float:
    return 4 * (n + 16) * U


def assert_within(name: str, got: torch.Tensor, want: torch.Tensor, tol: torch.Tensor) -> None:
    got, want, tol = got.double(), want.double(), tol.double()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    bad = ~((got - want).abs() <= tol)
    if bool(bad.any()):
        at = tuple(int(i) for i in bad.nonzero()[0])
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} values off; first at {at}: {float(got[at])} "
                             f"for {float(want[at])}, {float((got[at] - want[at]).abs()):.3g} > {float(tol[at]):.3g}")


# ------------------------------------------------------------------------------------------ layer norm


def norm_reference(x, gamma, beta, eps, dy):
    """{name: (value, bound)} of y, dx, dgamma, dbeta; x and dy as rows."""
    t = x.dtype
    x, dy = (a.double().reshape(-1, a.shape[-1]) for a in (x, dy))
    n, c = x.shape
    g = torch.ones(c, device=x.device, dtype=torch.float64) if gamma is None else gamma.double()
    b = torch.zeros_like(g) if beta is None else beta.double()
    mean = x.mean(-1, keepdim=True)
    var = ((x - mean) ** 2).mean(-1, keepdim=True)
    rstd = (var + eps) ** -0.5
    xhat = (x - mean) * rstd
    y = xhat * g + b
    gy = dy * g
    m0, m1 = gy.mean(-1, keepdim=True), (gy * xhat).mean(-1, keepdim=True)
    dx = rstd * (gy - m0 - xhat * m1)
    # A row is summed by each thread over at most 32 values, then in a tree: under 64 roundings.
    s = acc(64)
    size = x.abs().amax(-1, keepdim=True)
    # mean: s |x|; variance: twice that error relative to the spread, and s of itself.
    e_mean = s * size
    e_xhat = e_mean * rstd + xhat.abs() * (s + 2 * e_mean * rstd)
    e_y = half(t) * y.abs() + e_xhat * g.abs() + 4 * U * (xhat.abs() * g.abs() + b.abs())
    a0, a1 = gy.abs().mean(-1, keepdim=True), (gy.abs() * xhat.abs()).mean(-1, keepdim=True)
    e_rstd = s + 2 * e_mean * rstd
    e_m1 = s * a1 + (gy.abs() * e_xhat).mean(-1, keepdim=True)
    e_dx = half(t) * dx.abs() + rstd * (s * a0 + e_xhat * m1.abs() + xhat.abs() * e_m1) + \
        (e_rstd + 8 * U) * rstd * (gy.abs() + a0 + xhat.abs() * a1)
    tw = torch.float32 if gamma is None else gamma.dtype
    dg, db = (dy * xhat).sum(0), dy.sum(0)
    e_dg = half(tw) * dg.abs() + acc(n) * (dy * xhat).abs().sum(0) + (dy.abs() * e_xhat).sum(0)
    e_db = half(tw) * db.abs() + acc(n) * dy.abs().sum(0)
    f, fw = floor(t), floor(tw)
    return {"y": (y, e_y + f), "dx": (dx, e_dx + f), "dgamma": (dg, e_dg + fw), "dbeta": (db, e_db + fw)}


# ------------------------------------------------------------------------------------------- attention


def visible(n, lq, lk, causal, q_lens, k_lens, device):
    ql = torch.full((n,), lq) if q_lens is None else q_lens.cpu().long().clamp(0, lq)
    kl = torch.full((n,), lk) if k_lens is None else k_lens.cpu().long().clamp(0, lk)
    i, j = torch.arange(lq)[None, :, None], torch.arange(lk)[None, None, :]
    ql, kl = ql[:, None, None], kl[:, None, None]
    see = (i < ql) & (j < kl)
    if causal:
        see &= j <= i + kl - ql
    return see.to(device), (i < ql).to(device)[..., 0], (j < kl).to(device)[:, 0]


def attention_reference(q, k, v, dout, scale=None, causal=False, q_lens=None, k_lens=None, value=None):
    """{name: (value, bound)} of out, lse, dq, dk, dv. Rows behind the lengths are cut out before any arithmetic."""
    t = q.dtype
    lead = q.shape[:-3]
    q, k, v, dout = (x.reshape(-1, *x.shape[-3:]).transpose(1, 2).double() for x in (q, k, v, dout))
    n, h, lq, hd = q.shape
    hk, lk = k.shape[1], k.shape[2]
    rep = h // hk
    scale = hd**-0.5 if scale is None else scale
    see, q_in, k_in = visible(n, lq, lk, causal, q_lens, k_lens, q.device)
    used = see.any(-1)  # queries that see something
    q, dout = (torch.where(used[:, None, :, None], x, 0.0) for x in (q, dout))
    k, v = (torch.where(k_in[:, None, :, None], x, 0.0).repeat_interleave(rep, 1) for x in (k, v))
    see = see[:, None]
    z = (q @ k.transpose(-1, -2) * scale).masked_fill(~see, -math.inf)
    lse = torch.logsumexp(z, -1)
    p = torch.where(see, (z - torch.where(lse == -math.inf, 0.0, lse)[..., None]).exp(), 0.0)
    out = p @ v
    dp = dout @ v.transpose(-1, -2)
    D = (dout * out).sum(-1, keepdim=True)
    ds = p * (dp - D)
    dq, dk, dv = ds @ k * scale, ds.transpose(-1, -2) @ q * scale, p.transpose(-1, -2) @ dout
    # Bounds. A score is off by acc(hd) of its magnitude sum, and P relatively by twice that (its sum too); its
    # exponential by 2^-20 (approximations of 2^x and of the sum's reciprocal, and the score's own rounding). 16-bit
    # kernels round P and dS to the type before the second product: half a step, of the smallest one below the type's
    # normal range (P relative to its row's maximum or sum, so a floor on P itself).
    ht, fl = half(t), floor(t)
    mag = q.abs() @ k.abs().transpose(-1, -2) * abs(scale)
    es = acc(hd) * mag
    top = torch.where(see, es + 2 * U * z.abs().nan_to_num(0, 0, 0), 0.0)
    worst = top.amax(-1, keepdim=True)
    ep = (top + worst + 2.0**-20 + acc(lk)) * p  # of P in fp32
    e_out = ht * out.abs() + (ht * p + fl * see + ep) @ v.abs() + acc(lk) * (p @ v.abs())
    e_lse = worst[..., 0] + 2.0**-20 + acc(lk) + 4 * U * lse.abs().nan_to_num(0, 0, 0)
    e_dp = acc(hd) * (dout.abs() @ v.abs().transpose(-1, -2))
    e_D = (dout.abs() * (e_out + acc(hd) * out.abs())).sum(-1, keepdim=True)
    e_ds = ht * ds.abs() + fl * see + ep * (dp - D).abs() + p * (e_dp + e_D + 4 * U * (dp.abs() + D.abs()))
    w = abs(scale)
    e_dq = ht * dq.abs() + w * (e_ds @ k.abs()) + acc(lk) * w * (ds.abs() @ k.abs())
    e_dk = w * (e_ds.transpose(-1, -2) @ q.abs()) + acc(lq * rep) * w * (ds.abs().transpose(-1, -2) @ q.abs())
    e_dv = (ht * p + fl * see + ep).transpose(-1, -2) @ dout.abs() + acc(lq * rep) * (p.transpose(-1, -2) @ dout.abs())

    def shared(x):
        return x.unflatten(1, (hk, rep)).sum(2)

    dk, dv, e_dk, e_dv = shared(dk), shared(dv), shared(e_dk), shared(e_dv)
    e_dk, e_dv = e_dk + ht * dk.abs(), e_dv + ht * dv.abs()
    def tokens(x):
        return x.transpose(1, 2).reshape(*lead, x.shape[2], x.shape[1], hd)

    res = {m: (tokens(a), tokens(e) + fl)
           for m, a, e in (("out", out, e_out), ("dq", dq, e_dq), ("dk", dk, e_dk), ("dv", dv, e_dv))}
    res["lse"] = (lse, e_lse)
    return res


# ----------------------------------------------------------------------------------------- dropout-add


def philox_words(seed: int, offset: int, first: int, n: int) -> torch.Tensor:
    """Words ``first .. first + n`` of the stream (Philox-4x32-10, Salmon et al. 2011), in Python integers' arithmetic
    on torch int64: key = seed, counter = (index // 4, offset)."""
    low = 0xFFFFFFFF
    e = torch.arange(first, first + n)
    b = e // 4
    c = [b & low, b >> 32, torch.full_like(b, offset & low), torch.full_like(b, (offset >> 32) & low)]
    k = [seed & low, (seed >> 32) & low]
    for _ in range(10):
        p0, p1 = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [((p1 >> 32) & low) ^ c[1] ^ k[0], p1 & low, ((p0 >> 32) & low) ^ c[3] ^ k[1], p0 & low]
        k = [(k[0] + 0x9E3779B9) & low, (k[1] + 0xBB67AE85) & low]
    return torch.stack(c, -1).gather(-1, (e % 4)[:, None])[:, 0]


def keep_mask(shape, p: float, rng: torch.Tensor) -> torch.Tensor:
    seed, offset = (int(x) for x in rng.tolist())
    return (philox_words(seed, offset, 0, math.prod(shape)) >= round(p * 2.0**32)).view(shape)
