"""What AdamW and the norm of gradients refuse, and the tables of the 8-bit codes. No GPU needed."""

from __future__ import annotations

import ctypes
import math
from array import array

import pytest
import torch

from adamw_reference import M_TABLE, U_TABLE, codes, values
from unblend_b200 import _lib, training


def test_tables():
    """The description by bit patterns in the C header gives the same values."""
    for c in range(1, 128):
        assert float(torch.tensor((c + 889) << 20, dtype=torch.int32).view(torch.float32)) == float(M_TABLE[c])
    for c in range(1, 256):
        assert float(torch.tensor((c + 1777) << 19, dtype=torch.int32).view(torch.float32)) == float(U_TABLE[c])
    assert M_TABLE[127] == U_TABLE[255] == 1
    x = torch.randn(512, generator=torch.Generator().manual_seed(1)) * torch.linspace(0, 1, 512)
    # half a step, and near 0 the smallest code (1.25 or 1.125 of 2^-16)
    for table, step in ((M_TABLE, 2.0**-4), (U_TABLE, 2.0**-5)):
        y = x if table is M_TABLE else x.abs()
        c, top = codes(y, table)
        back = values(c, top, table)
        assert bool(((back - y).abs() <= step * y.abs() * 1.0001 + 1.25 * 2.0**-16 * top.repeat_interleave(256)).all())


def test_state_layout():
    params = [torch.zeros(3), torch.zeros(0), torch.zeros(16, 17), torch.zeros(256), torch.zeros(())]
    s = training.adamw_state(params)
    assert s.exp_avg.shape == (5 * 256,) and s.scales is None and s.exp_avg.dtype == torch.float32
    s8 = training.adamw_state(params, 8)
    assert s8.exp_avg.shape == (5 * 256,) and s8.scales.shape == (5, 2) and s8.exp_avg_sq.dtype == torch.uint8
    flat = torch.arange(5 * 256.0)
    views = training.adamw_views(params, flat)
    assert [v.shape for v in views] == [p.shape for p in params]
    assert views[0][0] == 0 and views[2][0, 0] == 256 and views[3][0] == 768 and views[4] == 1024
    assert training.adamw_moments(s)[0] is s.exp_avg


def test_states_are_saved_as_tuples(tmp_path):
    for bits in (32, 8):
        s = training.adamw_state([torch.zeros(300), torch.zeros(5)], bits)
        s.exp_avg[7] = 3
        torch.save(tuple(s), tmp_path / "state.pt")
        back = training.AdamWState(*torch.load(tmp_path / "state.pt", weights_only=True))
        assert all(a is b or torch.equal(a, b) for a, b in zip(s, back))
        assert training._check_state(back) == 3


def test_refuses():
    p, g = [torch.zeros(5), torch.zeros(2, 3)], [torch.zeros(5), torch.zeros(2, 3)]
    s = training.adamw_state(p)
    step = training.adamw_step
    one = torch.ones(1, dtype=torch.int64)
    for bad in (lambda: step(p[0], g, s, 1), lambda: step(p, g[0], s, 1), lambda: step(p, g[:1], s, 1),
                lambda: step([], [], s, 1), lambda: step(3, 4, s, 1), lambda: step(p, [g[0], g[1].t()], s, 1),
                lambda: step([p[0], p[1].t()], [g[0], g[1].t()], s, 1), lambda: step(p, [g[0], g[0]], s, 1),
                lambda: step([x.double() for x in p], g, s, 1), lambda: step(p, [x.double() for x in g], s, 1),
                lambda: step(p, [g[0], [1.0]], s, 1), lambda: step([p[0], 1.0], g, s, 1),
                lambda: step(p, [g[0], g[1].to_sparse()], s, 1),
                lambda: step(p, g, s, 0), lambda: step(p, g, s, -1), lambda: step(p, g, s, 1.0),
                lambda: step(p, g, s, True), lambda: step(p, g, s, one.int()), lambda: step(p, g, s, one.repeat(2)),
                lambda: step(p, g, s, 1 << 62), lambda: step(p, g, s, 1, lr=-1.0), lambda: step(p, g, s, 1, lr=math.nan),
                lambda: step(p, g, s, 1, lr=math.inf), lambda: step(p, g, s, 1, lr=1e19),
                lambda: step(p, g, s, 1, weight_decay=1e19), lambda: step(p, g, s, 1, lr=torch.ones(1).double()),
                lambda: step(p, g, s, 1, betas=(1.0, 0.9)), lambda: step(p, g, s, 1, betas=(0.9, -0.1)),
                lambda: step(p, g, s, 1, betas=0.9), lambda: step(p, g, s, 1, betas=(0.9,)),
                lambda: step(p, g, s, 1, eps=-1e-8), lambda: step(p, g, s, 1, eps=1e-40),
                lambda: step(p, g, s, 1, eps=1e31), lambda: step(p, g, s, 1, weight_decay=-0.1),
                lambda: step(p, g, s, 1, grad_scale=1.0), lambda: step(p, g, s, 1, grad_scale=torch.ones(2)),
                lambda: step(p, g, s, 1, grad_scale=torch.ones(1).half()),
                lambda: step(p, g, tuple(s), 1), lambda: step(p[:1], g[:1], s, 1),
                lambda: step(p, g, s._replace(exp_avg=s.exp_avg.half()), 1),
                lambda: step(p, g, s._replace(exp_avg=s.exp_avg[:256]), 1),
                lambda: step(p, g, s._replace(exp_avg=s.exp_avg_sq), 1),
                lambda: step(p, g, s._replace(exp_avg=torch.zeros(513)[1:]), 1),
                lambda: step(p, g, s._replace(scales=torch.zeros(2, 2)), 1),
                lambda: step(p, g, training.adamw_state(p, 8)._replace(scales=torch.zeros(2, 3)), 1),
                lambda: step(p, g, training.adamw_state(p, 8)._replace(scales=None), 1),
                lambda: training.adamw_state(p, 16), lambda: training.adamw_state([]),
                lambda: training.adamw_state([p[1].t()]), lambda: training.adamw_state(p[0]),
                lambda: training.adamw_views(p, torch.zeros(256)), lambda: training.adamw_moments(p)):
        with pytest.raises(ValueError):
            bad()
    conv = torch.zeros(2, 3, 4, 4).to(memory_format=torch.channels_last)
    with pytest.raises(ValueError, match="contiguous"):
        training.adamw_state([conv])
    neg = torch.zeros(5, dtype=torch.complex64).conj().imag
    for bad in (lambda: step([neg, p[1]], g, s, 1), lambda: step(p, [neg, g[1]], s, 1)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(ValueError, match="CUDA devices only"):
        step(p, g, s, 1)
    with pytest.raises(ValueError, match="CUDA devices only"):
        training.adamw_moments(training.adamw_state(p, 8))
    norm = training.grad_norm
    for bad in (lambda: norm([]), lambda: norm([None]), lambda: norm(g[0]), lambda: norm([g[1].t()]),
                lambda: norm([g[0].double()]), lambda: norm(g, 0.0), lambda: norm(g, -1.0), lambda: norm(g, math.nan),
                lambda: norm(g, math.inf), lambda: norm(g, 1e39), lambda: norm([1.0]), lambda: norm(g, "1")):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(ValueError, match="CUDA devices only"):
        norm(g, 1.0)


def _table(*rows):
    return array("q", [x for r in rows for x in r])


def test_entry_points_refuse_before_they_launch():
    lib = _lib.load()
    x = ctypes.create_string_buffer(1 << 16)
    p = (ctypes.addressof(x) + 15) & ~15
    good = _table((p, p + 4096, 10, 0))
    a = _lib.AdamWParams(1e-3, 0.9, 0.999, 1e-8, 0.01, 1)
    bad = _lib.ERR_INVALID

    def step(table=good, count=1, m=p, v=p + 8192, s=p, bits=32, dtype=0, grad=0, args=a):
        return lib.unblend_adamw_step(None if table is None else table.buffer_info()[0], count, m, v, s, bits, dtype,
                                      grad, None if args is None else ctypes.byref(args), None)

    def with_(**kw):
        b = _lib.AdamWParams(1e-3, 0.9, 0.999, 1e-8, 0.01, 1)
        for n, w in kw.items():
            setattr(b, n, w)
        return b

    for kw in (dict(table=None), dict(count=0), dict(count=-1), dict(m=None), dict(v=None), dict(m=p + 4),
               dict(v=p + 8), dict(bits=16), dict(bits=8, s=None), dict(bits=8, s=p + 4), dict(dtype=3), dict(grad=-1),
               dict(args=None), dict(args=with_(beta1=1.0)), dict(args=with_(beta2=-0.5)),
               dict(args=with_(beta1=math.nan)), dict(args=with_(eps=-1.0)), dict(args=with_(eps=math.inf)),
               dict(args=with_(eps=1e-40)), dict(args=with_(eps=math.nan)),
               dict(args=with_(lr=math.nan)), dict(args=with_(lr=1e19)), dict(args=with_(weight_decay=math.inf)), dict(args=with_(step=0)),
               dict(args=with_(step_device=p + 4)), dict(args=with_(lr_device=p + 2)),
               dict(args=with_(grad_scale=p + 1)), dict(table=_table((0, p, 10, 0))), dict(table=_table((p, 0, 10, 0))),
               dict(table=_table((p, p + 4096, 0, 0))), dict(table=_table((p, p + 4096, 10, -1))),
               dict(table=_table((p + 2, p + 4096, 10, 0))), dict(table=_table((p, p + 4098, 10, 0))),
               dict(table=_table((p, p + 4096, 1 << 39, 0)))):
        assert step(**kw) == bad, kw
    shared = _lib.ERR_OVERLAP
    assert step(_table((p, p + 4096, 10, 0), (p + 36, p + 4096, 10, 1)), 2) == shared
    assert step(_table((p, p + 36, 10, 0))) == shared
    assert step(_table((p, p + 4096, 1000, 0), (p + 8192, p, 10, 4)), 2) == shared
    assert lib.unblend_adamw_values(p, p, p, p, p, 0, None) == bad
    assert lib.unblend_adamw_values(p, p, p, p + 4, p, 1, None) == bad
    assert lib.unblend_adamw_values(None, p, p, p, p, 1, None) == bad
    n = ctypes.c_longlong(-1)
    assert lib.unblend_grad_norm_workspace(1, ctypes.byref(n)) == 0 and n.value >= 8
    assert lib.unblend_grad_norm_workspace(0, ctypes.byref(n)) == bad
    assert lib.unblend_grad_norm_workspace(1, None) == bad
    counts = (ctypes.c_int * 3)(1, 0, 0)
    t = good.buffer_info()[0]
    assert lib.unblend_grad_norm(None, counts, 1.0, p, p, p, None) == bad
    assert lib.unblend_grad_norm(t, None, 1.0, p, p, p, None) == bad
    assert lib.unblend_grad_norm(t, counts, 1.0, None, p, p, None) == bad
    assert lib.unblend_grad_norm(t, counts, 1.0, p, p, None, None) == bad
    assert lib.unblend_grad_norm(t, counts, 0.0, p, p, p, None) == bad
    assert lib.unblend_grad_norm(t, counts, math.nan, p, p, p, None) == bad
    assert lib.unblend_grad_norm(t, (ctypes.c_int * 3)(-1, 1, 0), 1.0, p, p, p, None) == bad
    odd = _table((0, p + 2, 10, 0))
    assert lib.unblend_grad_norm(odd.buffer_info()[0], counts, 1.0, p, p, p, None) == bad


def test_param_struct_layout(tmp_path):
    from test_capi import test_param_struct_layout_matches_c

    test_param_struct_layout_matches_c(tmp_path, _lib.AdamWParams, "UnblendAdamWParams")
