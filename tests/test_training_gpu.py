"""The training operators on the GPU against their 64-bit definitions (bounds: ``training_reference``)."""

from __future__ import annotations

import math

import pytest
import torch

from training_reference import (acc, assert_within, attention_reference, floor, half, keep_mask, norm_reference,
                                philox_words)
from unblend_b200 import _lib, training

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rand(*shape, g, t=F32, scale=1.0, shift=0.0):
    return (torch.randn(*shape, device="cuda", generator=g) * scale + shift).to(t)


def _check(res, got):
    for name, (want, tol) in res.items():
        if name in got:
            assert_within(name, got[name].reshape(want.shape), want, tol)


# ------------------------------------------------------------------------------------------ layer norm


def _norm_case(x, gamma, beta, dy, eps=1e-5):
    y, stats = training.layer_norm_forward(x, gamma, beta, eps)
    dx, dg, db = training.layer_norm_backward(dy, x, stats, gamma)
    assert y.dtype == dx.dtype == x.dtype and y.is_contiguous() and dx.is_contiguous()
    _check(norm_reference(x, gamma, beta, eps, dy), {"y": y, "dx": dx, "dgamma": dg, "dbeta": db})
    return y, dx, dg, db


@pytest.mark.parametrize("cols", [1, 7, 32, 250, 256, 264, 512, 513, 1000, 1024, 1032, 2047, 5003, 8192, 8201])
@pytest.mark.parametrize("t,tw", [(F32, F32), (BF16, F32), (BF16, BF16), (F16, F16)])
def test_norm_widths_and_types(t, tw, cols):
    g = _gen(cols)
    for rows in (1, 5, 333):
        x, dy = _rand(rows, cols, g=g, t=t, scale=2.0, shift=0.5), _rand(rows, cols, g=g, t=t)
        gamma, beta = _rand(cols, g=g, t=tw, scale=0.3, shift=1.0), _rand(cols, g=g, t=tw)
        _norm_case(x, gamma, beta, dy)


@pytest.mark.parametrize("t", [F32, BF16])
def test_norm_many_rows(t):
    g = _gen(1)
    x, dy = _rand(20011, 96, g=g, t=t), _rand(20011, 96, g=g, t=t)
    _norm_case(x, _rand(96, g=g), _rand(96, g=g), dy)
    x, dy = _rand(3001, 1200, g=g, t=t), _rand(3001, 1200, g=g, t=t)
    _norm_case(x, _rand(1200, g=g), _rand(1200, g=g), dy)


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("cols", [96, 1100])
def test_norm_strides(t, cols):
    g = _gen(2)
    big, other = _rand(4, 9, 7, cols + 5, g=g, t=t), _rand(4, 9, 7, cols, g=g, t=t)
    gamma, beta = _rand(cols, g=g), _rand(cols, g=g)
    pick = {
        "wide rows": (big[..., :cols], other), "off by one": (big[..., 1:cols + 1], other),
        "slice of both": (big[:, 2:7, :, 3:cols + 3], other[:, 2:7]),
        "transposed": (big[..., :cols].transpose(0, 1), other.transpose(0, 1)),
        "expanded gradient": (other, torch.ones((), device="cuda", dtype=t).expand(other.shape)),
        "expanded rows": (other[:1].expand(4, 9, 7, cols), other), "last axis strided": (big[..., :cols], other),
        "one row": (other[0, 0, 0], other[1, 1, 1]),
    }
    for x, dy in pick.values():
        _norm_case(x, gamma, beta, dy)
    cm = _rand(cols, 40, g=g, t=t).t()
    _norm_case(cm, gamma, beta, _rand(40, cols, g=g, t=t))


def test_norm_without_weights():
    g = _gen(3)
    x, dy = _rand(50, 300, g=g), _rand(50, 300, g=g)
    for gamma, beta in ((None, None), (_rand(300, g=g), None), (None, _rand(300, g=g))):
        _norm_case(x, gamma, beta, dy)
    y, stats = training.layer_norm_forward(x)
    dx, dg, db = training.layer_norm_backward(dy, x, stats, None, weight_grads=False)
    assert dg is None and db is None
    _check(norm_reference(x, None, None, 1e-5, dy), {"dx": dx})


def test_norm_hard_rows():
    """Constant rows, a mean far above the spread, tiny and huge values; NaN and infinities stay in their row."""
    g = _gen(4)
    x = _rand(9, 700, g=g)
    x[0] = 3.0
    x[1] = 0.0
    x[2] += 1000.0
    x[3] *= 1e-6
    x[4] *= 1e15
    gamma, beta, dy = _rand(700, g=g), _rand(700, g=g), _rand(9, 700, g=g)
    clean = _norm_case(x, gamma, beta, dy)
    assert torch.equal(clean[0][1], beta)
    x[6, 13], x[7, 5] = math.nan, math.inf
    y, stats = training.layer_norm_forward(x, gamma, beta)
    dx, _, _ = training.layer_norm_backward(dy, x, stats, gamma)
    keep = torch.tensor([0, 1, 2, 3, 4, 5, 8], device="cuda")
    assert torch.equal(y[keep], clean[0][keep]) and torch.equal(dx[keep], clean[1][keep])
    assert y[6].isnan().all() and y[7].isnan().all() and dx[6].isnan().all()


def test_norm_empty():
    x = torch.zeros(0, 5, 16, device="cuda")
    y, stats = training.layer_norm_forward(x, torch.ones(16, device="cuda"))
    dx, dg, db = training.layer_norm_backward(y, x, stats, torch.ones(16, device="cuda"))
    assert y.shape == dx.shape == x.shape and not dg.any() and not db.any()


# ----------------------------------------------------------------------------------------- dropout-add


def _drop_case(x, p, rng, residual, scale, dy):
    keep = keep_mask(x.shape, p, rng).to(x.device)
    f = 1 / (1 - p) if p < 1 else 0.0
    s = torch.ones(x.shape[-1], device="cuda", dtype=torch.float64) if scale is None else scale.double()
    y = training.dropout_add_forward(x, p, rng, residual, scale)
    dx, ds = training.dropout_add_backward(dy, x, p, rng, scale)
    assert y.is_contiguous() and dx.is_contiguous() and dx.dtype == x.dtype
    xd = torch.where(keep, x.double(), 0.0) * f
    branch = s * xd
    r = torch.zeros_like(xd) if residual is None else residual.double()
    # Four fp32 roundings (1 / (1 - p), its product, the scale's product, the sum), then the type's.
    assert_within("y", y, r + branch, half(y.dtype) * (r + branch).abs() + 4 * half(F32) * (r.abs() + branch.abs()) + floor(y.dtype))
    dd = torch.where(keep, dy.double(), 0.0) * f
    assert_within("dx", dx, s * dd, (half(x.dtype) + 4 * half(F32)) * (s * dd).abs() + floor(x.dtype))
    if scale is None:
        assert ds is None
    else:
        terms = torch.where(keep, dd * x.double(), 0.0).flatten(0, -2)
        want = terms.sum(0)
        assert ds.dtype == scale.dtype
        assert_within("dscale", ds, want, half(ds.dtype) * want.abs() + acc(len(terms)) * terms.abs().sum(0) + floor(ds.dtype))
    assert torch.equal(y, training.dropout_add_forward(x, p, rng, residual, scale))
    return y, dx, ds


@pytest.mark.parametrize("cols", [1, 3, 32, 33, 124, 125, 256, 1000, 2056, 4099])
@pytest.mark.parametrize("t,tr,tw", [(F32, F32, F32), (BF16, F32, F32), (BF16, BF16, BF16), (F16, F16, F32),
                                     (F16, F32, F16)])
def test_dropout_widths_and_types(t, tr, tw, cols):
    g = _gen(cols)
    rng = torch.randint(-(1 << 62), 1 << 62, (2,), device="cuda", generator=g)
    for rows, p in ((1, 0.3), (97, 0.1), (2, 0.5)):
        x, r, dy = (_rand(rows, cols, g=g, t=a) for a in (t, tr, tr))
        _drop_case(x, p, rng, r, _rand(cols, g=g, t=tw), dy)
    _drop_case(x, 0.2, rng, r, None, dy)
    _drop_case(x, 0.2, rng, None, None, dy)


def test_dropout_many_rows():
    g = _gen(5)
    for cols in (64, 61):
        x, r, dy = (_rand(30011, cols, g=g, t=a) for a in (BF16, F32, F32))
        _drop_case(x, 0.1, torch.tensor([7, 9], device="cuda"), r, _rand(cols, g=g), dy)


def test_dropout_extremes():
    """p of 0 and 1, probabilities next to them; a dropped element adds nothing, whatever it holds."""
    g = _gen(6)
    rng = torch.tensor([123, 456], device="cuda")
    for cols in (64, 61):
        x, r, dy = (_rand(40, cols, g=g) for _ in range(3))
        s = _rand(cols, g=g)
        for p in (0.0, 1.0, 1e-12, 1 - 1e-12, 1 - 2.0**-20):
            _drop_case(x, p, rng, r, s, dy)
        y, dx, ds = _drop_case(x, 1.0, rng, r, s, dy)
        assert torch.equal(y, r) and not dx.any() and not ds.any()
        keep = keep_mask(x.shape, 0.5, rng).cuda()
        x2, dy2 = torch.where(keep, x, math.inf), torch.where(keep, dy, math.nan)
        y = training.dropout_add_forward(x2, 0.5, rng, r, s)
        dx, ds = training.dropout_add_backward(dy2, x2, 0.5, rng, s)
        clean = training.dropout_add_backward(dy, x, 0.5, rng, s)
        assert torch.equal(y, training.dropout_add_forward(x, 0.5, rng, r, s))
        assert torch.equal(dx, clean[0]) and torch.equal(ds, clean[1])


@pytest.mark.parametrize("cols", [64, 61])
def test_dropout_strides(cols):
    """The mask goes by the row-major element number, not by the layout."""
    g = _gen(7)
    rng = torch.tensor([5, 6], device="cuda")
    big = _rand(3, 8, 5, cols + 3, g=g, t=BF16)
    r, dy = _rand(3, 8, 5, cols + 8, g=g), _rand(3, 8, 5, cols, g=g)
    s = _rand(cols, g=g)
    for x, res, d in ((big[..., :cols], r[..., :cols], dy), (big[..., 1:cols + 1], r[..., 8:], dy),
                      (big[:, 2:5, :, :cols], r[:, 2:5, :, :cols], dy[:, 1:4]),
                      (big[..., :cols].transpose(0, 2), r[..., :cols].transpose(0, 2), dy.transpose(0, 2)),
                      (big[:1, ..., :cols].expand(3, 8, 5, cols), r[..., :cols],
                       torch.ones((), device="cuda").expand(3, 8, 5, cols))):
        _drop_case(x, 0.25, rng, res, s, d)


@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("cols", [8, 64, 520, 4096])
def test_dropout_aligned_slices(cols, t):
    """Rows of 16-byte chunks with gaps between them, in one tensor or in all."""
    g = _gen(cols)
    rng = torch.tensor([8, 1 << 40], device="cuda")
    x, r, dy = (_rand(70, 3, cols + 16, g=g, t=a)[..., 8:-8] for a in (t, F32, F32))
    s = _rand(cols, g=g)
    _drop_case(x, 0.25, rng, r, s, dy)
    _drop_case(x, 0.25, rng, r.contiguous(), s, dy.contiguous())
    _drop_case(x.contiguous(), 0.25, rng, r, None, dy)


@pytest.mark.parametrize("cols", [1 << 22, (1 << 22) + 8, (1 << 22) + 5])
def test_dropout_very_wide_rows(cols):
    g = _gen(12)
    x, r, dy = (_rand(2, cols, g=g, t=a) for a in (BF16, F32, F32))
    _drop_case(x, 0.1, torch.tensor([3, 4], device="cuda"), r, _rand(cols, g=g), dy)


def test_dropout_keep_rate_and_streams():
    x = torch.ones(4000, 1000, device="cuda")
    seen = []
    for rng in ((1, 0), (1, 1), (2, 0), (1 + (1 << 32), 0), (1, 1 << 32)):
        y = training.dropout_add_forward(x, 0.3, torch.tensor(rng, device="cuda"))
        rate = float((y != 0).double().mean())
        assert abs(rate - 0.7) < 6 * math.sqrt(0.21 / x.numel())  # six standard deviations
        seen.append(y != 0)
    for a in range(len(seen)):
        for b in range(a):
            both = float((seen[a] & seen[b]).double().mean())  # independent masks: 0.49
            assert abs(both - 0.49) < 6 * math.sqrt(0.49 * 0.51 / x.numel())


def test_dropout_past_32_bits():
    """Elements behind number 2^32 draw their own words: the last rows of a tensor of 2^32 + 2^22 elements."""
    rows, cols = (1 << 18) + 256, 1 << 14
    x = torch.ones(1, cols, device="cuda", dtype=F16).expand(rows, cols)
    y = training.dropout_add_forward(x, 0.5, torch.tensor([11, 12], device="cuda"))
    for row in (0, (1 << 18) - 1, 1 << 18, rows - 1):
        want = philox_words(11, 12, row * cols, cols) >= 1 << 31
        assert torch.equal(y[row].cpu() != 0, want), row


# ------------------------------------------------------------------------------------------- attention


def _attn(lq, lk, h, hk, hd, t, n=2, seed=0, scale=1.0):
    g = _gen(seed)
    return (_rand(n, lq, h, hd, g=g, t=t, scale=scale), _rand(n, lk, hk, hd, g=g, t=t, scale=scale),
            _rand(n, lk, hk, hd, g=g, t=t), _rand(n, lq, h, hd, g=g, t=t))


def _attn_case(q, k, v, dout, **kw):
    out, lse = training.attention_forward(q, k, v, **kw)
    dq, dk, dv = training.attention_backward(dout, q, k, v, out, lse, **kw)
    torch.cuda.synchronize()
    assert _lib.error_flag() == 0
    assert all(x.is_contiguous() and x.dtype == q.dtype for x in (out, dq, dk, dv))
    got = {"out": out, "dq": dq, "dk": dk, "dv": dv}
    ref = attention_reference(q, k, v, dout, **kw)
    want, tol = ref.pop("lse")
    assert torch.equal(lse == -math.inf, want == -math.inf)
    fin = want != -math.inf
    assert_within("lse", lse[fin], want[fin], tol[fin])
    _check(ref, got)
    again = training.attention_forward(q, k, v, **kw)
    assert torch.equal(again[0], out) and torch.equal(again[1], lse)
    for a, b in zip(training.attention_backward(dout, q, k, v, out, lse, **kw), (dq, dk, dv)):
        assert torch.equal(a, b)
    return got


LENGTHS = [(1, 1), (1, 300), (300, 1), (5, 63), (64, 64), (65, 129), (128, 128), (129, 127), (200, 513), (257, 100)]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("lq,lk", LENGTHS)
def test_attention_lengths(lq, lk, t, causal):
    _attn_case(*_attn(lq, lk, 2, 2, 64, t, seed=lq + lk), causal=causal)


@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("hd", [1, 3, 8, 16, 20, 40, 48, 72, 80, 96, 100, 120, 128])
def test_attention_head_dims(hd, t):
    _attn_case(*_attn(150, 170, 2, 2, hd, t, seed=hd))
    _attn_case(*_attn(150, 170, 2, 1, hd, t, seed=hd), causal=True)


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("h,hk,hd", [(6, 2, 64), (4, 1, 128), (8, 8, 32), (5, 5, 64), (12, 3, 48)])
def test_attention_shared_heads(h, hk, hd, t):
    for causal in (False, True):
        _attn_case(*_attn(140, 260, h, hk, hd, t), causal=causal)
    _attn_case(*_attn(1, 700, h, hk, hd, t))


@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("hd", [48, 64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_ragged(causal, hd, t):
    """Lengths of zero, one, full, next to tile borders and outside the range (clamped); padding holds NaN."""
    ql = torch.tensor([0, 1, 64, 65, 200, 128, 300, 200, 13, -5], device="cuda", dtype=torch.int32)
    kl = torch.tensor([50, 0, 63, 64, 256, 999, 257, 1, 129, 60], device="cuda", dtype=torch.int32)
    q, k, v, dout = _attn(200, 257, 2, 1, hd, t, n=10)
    for b in range(10):
        a, c = min(max(int(ql[b]), 0), 200), min(max(int(kl[b]), 0), 257)
        q[b, a:], dout[b, a:], k[b, c:], v[b, c:] = math.nan, math.inf, math.nan, math.inf
        if causal and a > c:  # queries in front that see no key
            q[b, : a - c] = math.nan
            dout[b, : a - c] = math.nan
    for kw in (dict(q_lens=ql, k_lens=kl), dict(k_lens=kl), dict(q_lens=ql)):
        qq, dd = (q, dout) if "q_lens" in kw and "k_lens" in kw else (q.nan_to_num(0.5), dout.nan_to_num(0.5, 0.5, 0.5))
        kk, vv = (k, v) if "k_lens" in kw else (k.nan_to_num(0.5), v.nan_to_num(0.5, 0.5, 0.5))
        if "q_lens" in kw and "k_lens" not in kw:
            for b in range(10):
                qq = qq.clone()
                qq[b, min(max(int(ql[b]), 0), 200):] = math.nan
        got = _attn_case(qq, kk, vv, dd, causal=causal, **kw)
        for b in range(10):
            c = min(max(int(kl[b]), 0), 257) if "k_lens" in kw else 257
            assert not got["dk"][b, c:].any() and not got["dv"][b, c:].any()


@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("h,hk,hd", [(2, 2, 64), (4, 1, 64), (3, 3, 128), (4, 2, 128), (2, 1, 40), (3, 3, 72)])
def test_attention_one_tile(h, hk, hd, t):
    """Sequences of up to 64 queries and keys, which 16-bit types do in one kernel: lengths, layouts, empty rows."""
    for lq, lk in ((17, 33), (64, 64), (62, 62), (63, 9), (33, 64), (16, 48), (32, 32), (17, 31), (1, 30), (31, 1), (16, 16)):
        for causal in (False, True):
            _attn_case(*_attn(lq, lk, h, hk, hd, t, seed=lq + hd), causal=causal)
    # [outer, inner = bands, tokens]: rows, heads and sequences apart, and gaps between rows.
    g = _gen(hd)
    x = _rand(3, 50, 5, h + 2 * hk, hd + 8, g=g, t=t)[..., :hd].transpose(1, 2)
    q, k, v = x.split((h, hk, hk), -2)
    _attn_case(q, k, v, _rand(3, 50, 5, h, hd, g=g, t=t).transpose(1, 2), scale=0.2)
    ql = torch.tensor([0, 1, 15, 16, 17, 64, 99, 40, 60, -3], device="cuda", dtype=torch.int32)
    kl = torch.tensor([20, 0, 16, 64, 1, 63, 50, 9, 0, 60], device="cuda", dtype=torch.int32)
    for causal in (False, True):
        q, k, v, dout = _attn(60, 64, h, hk, hd, t, n=10)
        for b in range(10):
            a, c = min(max(int(ql[b]), 0), 60), min(max(int(kl[b]), 0), 64)
            q[b, a:], dout[b, a:], k[b, c:], v[b, c:] = math.nan, math.inf, math.nan, math.inf
            if c == 0 or (causal and a > c):  # queries that see no key
                q[b, : a - c] = math.nan
                dout[b, : a - c] = math.nan
        got = _attn_case(q, k, v, dout, causal=causal, q_lens=ql, k_lens=kl)
        for b in range(10):
            a, c = min(max(int(ql[b]), 0), 60), min(max(int(kl[b]), 0), 64)
            assert not got["out"][b, a:].any() and not got["dq"][b, a:].any()
            assert not got["dk"][b, c:].any() and not got["dv"][b, c:].any()


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("h,hk,hd", [(2, 2, 64), (6, 2, 48), (2, 1, 128)])
def test_attention_half_tile_ragged(h, hk, hd, t, causal):
    """Sequences of up to 32 queries and keys with lengths of their own; padding holds NaN."""
    ql = torch.tensor([0, 1, 15, 16, 17, 31, 40, 30, 5, -1], device="cuda", dtype=torch.int32)
    kl = torch.tensor([20, 0, 16, 32, 1, 29, 50, 9, 0, 17], device="cuda", dtype=torch.int32)
    q, k, v, dout = _attn(31, 32, h, hk, hd, t, n=10)
    for b in range(10):
        a, c = min(max(int(ql[b]), 0), 31), min(max(int(kl[b]), 0), 32)
        q[b, a:], dout[b, a:], k[b, c:], v[b, c:] = math.nan, math.inf, math.nan, math.inf
        if c == 0 or (causal and a > c):  # queries that see no key
            q[b, : a - c] = math.nan
            dout[b, : a - c] = math.nan
    _attn_case(q, k, v, dout, causal=causal, q_lens=ql, k_lens=kl)


@pytest.mark.parametrize("t", [BF16, F16])
def test_attention_one_tile_far_rows(t):
    """Rows of a short sequence 2^24 and more elements apart."""
    buf = torch.empty(40 * ((1 << 24) + 8), device="cuda", dtype=t)
    for stride in ((1 << 24) - 8, 1 << 24):
        q = buf.as_strided((1, 40, 2, 64), (0, stride, 64, 1))
        q.copy_(_rand(1, 40, 2, 64, g=_gen(4), t=t))
        _attn_case(q, q, q, q)


@pytest.mark.parametrize("t", [F32, BF16, F16])
def test_attention_layouts(t):
    """One packed projection, the two token axes of an axial model, rows that TMA cannot address, expanded heads."""
    g = _gen(8)
    o, length, bands, h, hd = 2, 70, 9, 3, 64
    x = _rand(o, length, bands, 3, h, hd, g=g, t=t)
    dout = _rand(o, length, bands, h, hd, g=g, t=t)
    q, k, v = x.unbind(3)
    _attn_case(q, k, v, dout)  # along the bands: [outer, inner = time, bands]
    _attn_case(*(y.transpose(1, 2) for y in (q, k, v, dout)))  # along time: [outer, inner = bands, time]
    _attn_case(*(y.transpose(1, 2) for y in (q, k, v, dout)), causal=True, scale=0.3)
    flat = [y.flatten(0, 1) for y in (q.contiguous(), k.contiguous(), v.contiguous(), dout)]
    _attn_case(*flat)
    hm = [y.transpose(1, 2).contiguous().transpose(1, 2) for y in flat]  # heads in front of tokens in memory
    _attn_case(*hm)
    odd = _rand(2, 100, 3 * h * hd + 1, g=g, t=t)[..., 1:].unflatten(-1, (3, h, hd)).unbind(2)
    _attn_case(*odd, _rand(2, 100, h, hd, g=g, t=t))
    shift = _rand(2 * 100 * h * hd + 1, g=g, t=t)[1:].view(2, 100, h, hd)
    _attn_case(shift, shift, shift, shift)
    one = _rand(2, 100, 1, hd, g=g, t=t).expand(2, 100, h, hd)
    _attn_case(flat[0][:2, :, :, :], one, one, flat[3][:2])
    ones = torch.ones((), device="cuda", dtype=t).expand(flat[0].shape)
    _attn_case(flat[0], flat[1], flat[2], ones)
    cols = _rand(2, 100, h, hd * 2, g=g, t=t)[..., ::2]
    _attn_case(cols, cols, cols, cols)


@pytest.mark.parametrize("t", [F32, BF16, F16])
def test_attention_long_and_few(t):
    """Few queries over many keys and the other way round: the split axes."""
    _attn_case(*_attn(3, 5000, 2, 1, 64, t, n=1))
    _attn_case(*_attn(3000, 17, 2, 1, 64, t, n=1))
    _attn_case(*_attn(700, 900, 1, 1, 128, t, n=1), causal=True)
    kl = torch.tensor([2100], device="cuda", dtype=torch.int32)
    _attn_case(*_attn(1, 4100, 4, 2, 128, t, n=1), k_lens=kl)


@pytest.mark.parametrize("t", [F32, BF16, F16])
def test_attention_large_scores(t):
    """Scores of +-100 and more: one key takes nearly all of the weight, sums neither overflow nor vanish."""
    q, k, v, dout = _attn(130, 260, 1, 1, 64, t, scale=4.0)
    _attn_case(q, k, v, dout)
    _attn_case(q, k, v, dout, scale=-0.2)
    _attn_case(q, k, v, dout, scale=0.0)


@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("lq,lk,cut,h,hk,hd", [(60, 64, 31, 2, 2, 64), (50, 60, 20, 4, 2, 48), (64, 64, 63, 3, 3, 128),
                                               (150, 300, 130, 2, 1, 64), (33, 200, 100, 2, 1, 128)])
def test_attention_blocks_of_keys(lq, lk, cut, h, hk, hd, t):
    """Two blocks of keys, each with a backward call of its own from the joined output and lse: the gradients of the
    whole. The output in t is the joined one rounded, as the whole's is, so the whole's bounds hold; dq is a sum of two
    rounded results."""
    q, k, v, dout = _attn(lq, lk, h, hk, hd, t)
    ref = attention_reference(q, k, v, dout)
    out, lse = training.attention_forward(q, k, v)
    parts = [training.attention_backward(dout, q, k[:, s], v[:, s], out, lse) for s in (slice(0, cut), slice(cut, lk))]
    got = {"dk": torch.cat([x[1] for x in parts], 1), "dv": torch.cat([x[2] for x in parts], 1)}
    _check({n: ref[n] for n in got}, got)
    want, tol = ref["dq"]
    each = half(t) * sum(x[0].double().abs() for x in parts)
    assert_within("dq", parts[0][0].double() + parts[1][0].double(), want, tol + each + floor(t))


def test_attention_nan_stays_in_its_sequence():
    q, k, v, dout = _attn(100, 100, 2, 2, 64, BF16, n=3)
    clean = _attn_case(q, k, v, dout)
    k[1, 7, 1, 3] = math.nan
    out, lse = training.attention_forward(q, k, v)
    grads = training.attention_backward(dout, q, k, v, out, lse)
    for got, want in zip((out, *grads), (clean[n] for n in ("out", "dq", "dk", "dv"))):
        assert torch.equal(got[[0, 2]], want[[0, 2]]) and torch.equal(got[1, :, 0], want[1, :, 0])
    assert out[1, :, 1].isnan().all()


def test_attention_empty():
    z = torch.zeros(0, 5, 2, 16, device="cuda")
    assert training.attention(z, z, z).shape == z.shape
    q, k = torch.ones(2, 3, 2, 16, device="cuda"), torch.zeros(2, 0, 2, 16, device="cuda")
    out, lse = training.attention_forward(q, k, k)
    assert not out.any() and (lse == -math.inf).all()
    dq, dk, dv = training.attention_backward(q, q, k, k, out, lse)
    assert not dq.any() and dk.shape == k.shape == dv.shape
    k = torch.ones(2, 3, 2, 16, device="cuda")
    out, lse = training.attention_forward(q[:, :0], k, k)
    dq, dk, dv = training.attention_backward(q[:, :0], q[:, :0], k, k, out, lse)
    assert dq.shape == (2, 0, 2, 16) and not dk.any() and not dv.any()


@pytest.mark.parametrize("t", [F32, BF16])
def test_attention_strides_past_32_bits(t):
    """Rows more than 2^31 elements apart in one buffer (a slice of a long cache)."""
    far = (1 << 30) + 64
    buf = torch.empty(3 * far, device="cuda", dtype=t)
    k = buf.as_strided((4, 70, 1, 64), (far // 2 * 1, 128, 64, 1))
    v = buf.as_strided((4, 70, 1, 64), (far // 2 * 1, 128, 64, 1), 64)
    g = _gen(9)
    k.copy_(_rand(4, 70, 1, 64, g=g, t=t))
    v.copy_(_rand(4, 70, 1, 64, g=g, t=t))
    q, dout = _rand(4, 70, 1, 64, g=g, t=t), _rand(4, 70, 1, 64, g=g, t=t)
    _attn_case(q, k, v, dout)


# ----------------------------------------------------------------------- streams, graphs, autograd, block


def _step(s):
    """All three operators in both directions with plain calls."""
    y, stats = training.layer_norm_forward(s["x"], s["gamma"], s["beta"])
    h = y.view(2, -1, 3, 2, 64)
    q, k, v = h.unbind(2)
    out, lse = training.attention_forward(q, k, v, causal=True)
    z = training.dropout_add_forward(out.flatten(-2), 0.2, s["rng"], s["res"], s["scale"])
    do, dscale = training.dropout_add_backward(s["dz"], out.flatten(-2), 0.2, s["rng"], s["scale"])
    dq, dk, dv = training.attention_backward(do.view_as(out), q, k, v, out, lse, causal=True)
    dy = torch.stack((dq, dk, dv), 2).view_as(s["x"])
    dx, dg, db = training.layer_norm_backward(dy, s["x"], stats, s["gamma"])
    return z, dscale, dx, dg, db


def _step_inputs(seed, t=BF16, length=150):
    g = _gen(seed)
    return {"x": _rand(2, length, 384, g=g, t=t), "gamma": _rand(384, g=g), "beta": _rand(384, g=g),
            "rng": torch.tensor([seed, 3], device="cuda"), "res": _rand(2, length, 128, g=g),
            "scale": _rand(128, g=g), "dz": _rand(2, length, 128, g=g)}


@pytest.mark.parametrize("t", [F32, BF16])
def test_two_captured_graphs_replayed_in_turn(t):
    """Two graphs of the whole step replay in turn and at once on two streams; new inputs and masks are seen."""
    a, b = _step_inputs(1, t), _step_inputs(2, t)
    fresh = _step_inputs(3, t)
    want = {n: [x.clone() for x in _step(s)] for n, s in (("a", a), ("b", b), ("fresh", fresh))}
    graphs, outs = [], []
    for s in (a, b):
        _step(s)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_step(s))
        graphs.append(graph)
    for order in ((0, 1), (1, 0)):
        for n in order:
            graphs[n].replay()
        for n, name in ((0, "a"), (1, "b")):
            assert all(torch.equal(x, y) for x, y in zip(outs[n], want[name]))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for graph, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    for n, name in ((0, "a"), (1, "b")):
        assert all(torch.equal(x, y) for x, y in zip(outs[n], want[name]))
    for name in a:
        a[name].copy_(fresh[name])
    graphs[0].replay()
    assert all(torch.equal(x, y) for x, y in zip(outs[0], want["fresh"]))
    assert _lib.error_flag() == 0


def test_other_streams_at_once():
    cases = [_step_inputs(s, length=100 + 37 * s) for s in range(4)]
    want = [[x.clone() for x in _step(s)] for s in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = []
    for _ in range(3):
        got.append([])
        for s, st in zip(cases, streams):
            with torch.cuda.stream(st):
                got[-1].append(_step(s))
    torch.cuda.synchronize()
    for rep in got:
        for one, ref in zip(rep, want):
            assert all(torch.equal(x, y) for x, y in zip(one, ref))


def test_autograd_is_refused_while_capturing():
    x = torch.randn(4, 64, device="cuda", requires_grad=True)
    q = torch.randn(1, 4, 1, 64, device="cuda", requires_grad=True)
    rng = torch.zeros(2, device="cuda", dtype=torch.int64)
    calls = (lambda: training.layer_norm(x), lambda: training.attention(q, q, q), lambda: training.dropout_add(x, 0.1, rng))
    kept = [c() for c in calls]  # eager passes that hold the leaves
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for c in calls:
            with pytest.raises(RuntimeError, match="captured"):
                c()
        with torch.no_grad():
            y = training.layer_norm(x)
    graph.replay()
    assert torch.equal(y, kept[0])
    for k in kept:
        k.sum().backward()
    assert x.grad is not None and q.grad is not None


def _block(p, x, rng, lib):
    """Pre-norm attention block: x + scale * dropout(proj(attention(qkv(norm(x))))), 2 heads."""
    h = lib["norm"](x, p["gamma"], p["beta"])
    q, k, v = (h @ p["wqkv"]).unflatten(-1, (3, 2, -1)).unbind(-3)
    a = lib["attention"](q, k, v).flatten(-2) @ p["wo"]
    return lib["drop"](a, rng, x, p["scale"])


def test_block_gradients_against_the_formula_and_differences():
    """The operators together, through autograd, against a 64-bit block and against its differences."""
    g = _gen(10)
    d, p_drop = 96, 0.2
    rng = torch.tensor([77, 5], device="cuda")
    shapes = {"gamma": (d,), "beta": (d,), "wqkv": (d, 3 * d), "wo": (d, d), "scale": (d,)}
    par = {n: _rand(*s, g=g, scale=d**-0.5 if n.startswith("w") else 0.5) for n, s in shapes.items()}
    par["gamma"] += 1
    x, w = _rand(2, 75, d, g=g), _rand(2, 75, d, g=g)
    keep = keep_mask(x.shape, p_drop, rng).cuda().double() / (1 - p_drop)

    def norm64(x, gamma, beta):
        c = x - x.mean(-1, keepdim=True)
        return c * ((c * c).mean(-1, keepdim=True) + 1e-5) ** -0.5 * gamma + beta

    def attention64(q, k, v):
        z = torch.einsum("bihd,bjhd->bhij", q, k) * q.shape[-1] ** -0.5
        return torch.einsum("bhij,bjhd->bihd", z.softmax(-1), v)

    ref_ops = {"norm": norm64, "attention": attention64, "drop": lambda a, rng, x, s: x + s * keep * a}
    own_ops = {"norm": training.layer_norm, "attention": training.attention,
               "drop": lambda a, rng, x, s: training.dropout_add(a, p_drop, rng, x, s)}
    leaves = {**par, "x": x}
    own = {n: t.clone().requires_grad_() for n, t in leaves.items()}
    ref = {n: t.double().requires_grad_() for n, t in leaves.items()}
    y = _block(own, own["x"], rng, own_ops)
    y64 = _block(ref, ref["x"], rng, ref_ops)
    # fp32 throughout: products over at most 3 * 96 and sums over 150 rows, each relative to its magnitudes, which
    # exceed the results by less than 30 here: 4 (288 + 16) 2^-24 * 30 = 2.2e-3 of the largest value at worst, and a
    # hundredth of it for roundings that do not all point one way.
    tol = acc(288) * 30 / 100
    assert float((y - y64).abs().max()) < tol * float(y64.abs().max())
    (y * w).sum().backward()
    (y64 * w.double()).sum().backward()
    for n in leaves:
        assert float((own[n].grad - ref[n].grad).abs().max()) < tol * float(ref[n].grad.abs().max()), n
    # Directional differences of the 64-bit block: error of order step^2 plus 1e-16 / step.
    for n in leaves:
        dirn = torch.randn(leaves[n].shape, device="cuda", generator=g, dtype=torch.float64)

        def loss(step):
            moved = {m: (t.detach() + step * dirn if m == n else t.detach()) for m, t in ref.items()}
            return float((_block(moved, moved["x"], rng, ref_ops) * w.double()).sum())

        diff = (loss(1e-5) - loss(-1e-5)) / 2e-5
        mine = float((own[n].grad.double() * dirn).sum())
        size = float((own[n].grad.double() * dirn).abs().sum())
        assert abs(mine - diff) < tol * size + 1e-6 * abs(diff), (n, mine, diff)


def test_gradients_of_expanded_and_shared_inputs():
    """Leaves that are broadcast into the call, or given to it twice, get the sum of their uses' gradients."""
    g = _gen(11)
    x = _rand(1, 1, 64, g=g).requires_grad_()
    training.layer_norm(x.expand(3, 5, 64), None, None).square().sum().backward()
    want = torch.func.grad(lambda t: torch.nn.functional.layer_norm(t, (64,)).square().sum() * 15)(x.detach())
    assert torch.allclose(x.grad, want, atol=1e-4)
    kv = _rand(2, 40, 1, 64, g=g).requires_grad_()
    q = _rand(2, 40, 4, 64, g=g)
    w = _rand(2, 40, 4, 64, g=g)
    (training.attention(q, kv.expand(2, 40, 4, 64), kv.expand(2, 40, 4, 64)) * w).sum().backward()
    once = kv.detach().clone().requires_grad_()
    (training.attention(q, once, once) * w).sum().backward()
    assert torch.allclose(kv.grad, once.grad, atol=1e-4)
