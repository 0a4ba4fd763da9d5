"""What the rotary operators refuse, their frequencies and parameters. No GPU needed."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from rotary_reference import check_pi, exact_angle
from unblend_b200 import _lib, training


def test_exact_angles():
    assert check_pi()
    assert abs(exact_angle(1, 0.5) - 0.5) < 1e-15 and abs(exact_angle(4, 1.0) - (4 - 2 * math.pi)) < 1e-15


def test_frequencies():
    f = training.rotary_freqs(64)
    assert f.dtype == torch.float64 and f.shape == (32,)
    assert torch.allclose(f, torch.tensor([10000.0 ** (-2 * i / 64) for i in range(32)], dtype=torch.float64),
                          rtol=1e-15)
    assert torch.equal(training.rotary_freqs(64, factor=4.0), f / 4)
    b = training.rotary_freqs(64, factor=4.0, method="base")
    assert b[0] == 1 and math.isclose(float(b[-1]), float(f[-1]) / 4, rel_tol=1e-14)
    assert bool((b <= f).all()) and bool((b >= f / 4 * (1 - 1e-14)).all())
    p = training.rotary_freqs(64, factor=4.0, method="parts", trained_length=1024)
    turns = 1024 * f / (2 * math.pi)
    assert torch.equal(p[turns >= 32], f[turns >= 32]) and torch.equal(p[turns <= 1], f[turns <= 1] / 4)
    mid = (turns > 1) & (turns < 32)
    keep = (turns[mid] - 1) / 31
    assert mid.any() and torch.allclose(p[mid], f[mid] * keep + f[mid] / 4 * (1 - keep), rtol=1e-14)
    for m in ("linear", "base"):
        assert torch.equal(training.rotary_freqs(2, method=m), torch.ones(1, dtype=torch.float64))
        assert torch.equal(training.rotary_freqs(64, method=m), f)


def test_frequencies_refuse():
    for bad in (dict(dims=0), dict(dims=3), dict(dims=-2), dict(dims=4.0), dict(dims=4, base=0.0),
                dict(dims=4, base=math.inf), dict(dims=4, factor=0.5), dict(dims=4, factor=math.nan),
                dict(dims=4, method="other"), dict(dims=4, method="parts"),
                dict(dims=4, method="parts", trained_length=0), dict(dims=2, factor=2.0, method="base"),
                dict(dims=4, method="parts", trained_length=9, slow=2.0, fast=2.0)):
        with pytest.raises(ValueError):
            training.rotary_freqs(**bad)


def test_rotary_refuses():
    q, k, f = torch.zeros(2, 5, 4, 16), torch.zeros(2, 5, 2, 16), torch.ones(8)
    pos = torch.arange(5)
    for call in (training.rotary, training.rotary_forward, training.rotary_backward):
        for bad in (lambda: call(q[0], k, f), lambda: call(q, k[:1], f), lambda: call(q, k[:, :4], f),
                    lambda: call(q, k.half(), f), lambda: call(q, k[..., :8], f), lambda: call(q.double(), None, f),
                    lambda: call(q, k, None), lambda: call(q, k, f.half()), lambda: call(q, k, torch.ones(9)),
                    lambda: call(q, k, f[None]), lambda: call(q, k, [1.0]), lambda: call(q, k, f, pos[:4]),
                    lambda: call(q, k, f, pos.float()), lambda: call(q, k, f, pos[None]),
                    lambda: call(q, k, f, [0, 1, 2, 3, 4]), lambda: call(q, k, f, scale=math.inf),
                    lambda: call(q, k, f, scale=math.nan), lambda: call(q, k, f, scale=1e39),
                    lambda: call(torch.zeros(1, 1, 1, 257), None, f), lambda: call(torch.zeros(1, 1, 1, 0), None, f),
                    lambda: call(q, k, f.clone().requires_grad_()),
                    lambda: call(q.clone().requires_grad_(), k, f.clone().requires_grad_()), lambda: call([1.0], None, f),
                    lambda: call(torch.zeros(1, 1, 1, 1).expand(1 << 16, 1 << 15, 1, 1), None, f[:0])):
            with pytest.raises(ValueError):
                bad()
        with pytest.raises(ValueError, match="CUDA devices only"):
            call(q, k, f, pos)


def test_qk_norm_refuses():
    q, k, f, w = torch.zeros(2, 5, 4, 16), torch.zeros(2, 5, 2, 16), torch.ones(8), torch.ones(16)
    lens = torch.zeros(2, dtype=torch.int32)
    for call in (training.qk_norm_rotary, training.qk_norm_rotary_forward,
                 lambda *a, **kw: training.qk_norm_rotary_backward(*a[:2], *a, **kw)):
        for bad in (lambda: call(q, k, w[:8], w, f), lambda: call(q, k, w, w.half(), f),
                    lambda: call(q, k, w.double(), None, f), lambda: call(q, None, w, w, f),
                    lambda: call(q.half(), k.half(), w, w.half(), f), lambda: call(q, k, w, w, f, eps=-1.0),
                    lambda: call(q, k, w, w, f, eps=math.nan), lambda: call(q, k, w, w, f, lens=lens.long()),
                    lambda: call(q, k, w, w, f, lens=lens[:1]), lambda: call(q, k, w, w, f, lens=[5, 5]),
                    lambda: call(q, k, w, w, f.half()), lambda: call(q, k, w[None], w, f)):
            with pytest.raises(ValueError):
                bad()
        with pytest.raises(ValueError, match="CUDA devices only"):
            call(q, k, w, w, f, lens=lens)
    back = training.qk_norm_rotary_backward
    for bad in (lambda: back(q, None, q, k), lambda: back(q, k, q, None), lambda: back(None, k, q, k),
                lambda: back(q[:, :4], k, q, k), lambda: back(q.half(), k, q, k), lambda: back(q, q, q, k)):
        with pytest.raises(ValueError):
            bad()


def _params(**kw):
    p = _lib.RotaryParams()
    base = dict(dtype=_lib.DTYPE_BF16, outer=2, inner=1, length=10, heads=4, k_heads=2, hd=64, pairs=0, scale=1.0,
                eps=1e-6)
    for n, v in {**base, **kw}.items():
        setattr(p, n, v)
    return p


def test_entry_points_refuse_before_they_launch():
    lib = _lib.load()
    n = ctypes.c_longlong(-1)
    work = lib.unblend_qk_norm_rotary_grad_workspace
    assert work(ctypes.byref(_params()), ctypes.byref(n)) == 0 and n.value >= 2 * 64 * 4
    bad = _lib.ERR_INVALID
    x = ctypes.create_string_buffer(64)
    p = ctypes.addressof(x) & ~15
    wrong = (dict(dtype=3), dict(outer=0), dict(inner=0), dict(length=0), dict(heads=0), dict(k_heads=-1), dict(hd=0),
             dict(hd=257), dict(pairs=33), dict(pairs=-1), dict(pairs=4), dict(scale=math.nan), dict(scale=math.inf),
             dict(outer=1 << 16, inner=1 << 15), dict(outer=1 << 20, length=1 << 10, heads=4),
             dict(pairs=4, freqs=p + 2), dict(pairs=4, freqs=p + 4, freqs_f64=1), dict(positions=p + 4, positions_i64=1))
    for kw in wrong:
        q = ctypes.byref(_params(**kw))
        assert work(q, ctypes.byref(n)) == bad, kw
        assert lib.unblend_rotary(p, p, p, p, q, 0, None) == bad, kw
        assert lib.unblend_qk_norm_rotary_forward(p, p, p, p, q, None) == bad, kw
        assert lib.unblend_qk_norm_rotary_backward(p, p, p, p, p, p, None, None, None, q, None) == bad, kw
    q = ctypes.byref(_params())
    assert work(None, ctypes.byref(n)) == bad and work(q, None) == bad
    assert lib.unblend_rotary(None, p, p, p, q, 0, None) == bad
    assert lib.unblend_rotary(p, None, p, p, q, 0, None) == bad
    assert lib.unblend_rotary(p, p, p, None, q, 0, None) == bad
    assert lib.unblend_qk_norm_rotary_forward(p, p, None, p, q, None) == bad
    assert lib.unblend_qk_norm_rotary_backward(p, p, p, p, p, p, p, None, p, q, None) == bad
    assert lib.unblend_qk_norm_rotary_backward(p, p, p, p, p, p, p, p, None, q, None) == bad
    for kw in (dict(eps=-1.0), dict(eps=math.nan), dict(w_dtype=_lib.DTYPE_F16), dict(w_dtype=7)):
        assert lib.unblend_qk_norm_rotary_forward(p, p, p, p, ctypes.byref(_params(**kw)), None) == bad


def test_param_struct_layout(tmp_path):
    from test_capi import test_param_struct_layout_matches_c

    test_param_struct_layout_matches_c(tmp_path, _lib.RotaryParams, "UnblendRotaryParams")
