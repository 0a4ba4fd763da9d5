"""What the training operators refuse, their row layouts and workspaces, and the random stream. No GPU needed."""

from __future__ import annotations

import ctypes

import pytest
import torch

from training_reference import philox_words
from unblend_b200 import _lib, training


def test_norm_refuses():
    x = torch.zeros(4, 8)
    g = torch.ones(8)
    for bad in (lambda: training.layer_norm(x.double(), g, g), lambda: training.layer_norm(x, g[:7], g),
                lambda: training.layer_norm(x, g.half(), g), lambda: training.layer_norm(x.half(), g.half(), g),
                lambda: training.layer_norm(x, g, g, eps=-1.0), lambda: training.layer_norm(torch.zeros(3, 0)),
                lambda: training.layer_norm([1.0], g, g), lambda: training.layer_norm(x.to(torch.int32)),
                lambda: training.layer_norm_backward(x[:2], x, torch.zeros(4, 2)),
                lambda: training.layer_norm_backward(x, x, torch.zeros(3, 2)),
                lambda: training.layer_norm_backward(x.half(), x, torch.zeros(4, 2))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(ValueError, match="CUDA devices only"):
        training.layer_norm(x, g, g)


def test_dropout_refuses():
    x, rng = torch.zeros(4, 8), torch.zeros(2, dtype=torch.int64)
    for bad in (lambda: training.dropout_add(x, -0.1, rng), lambda: training.dropout_add(x, 1.5, rng),
                lambda: training.dropout_add(x, float("nan"), rng), lambda: training.dropout_add(x, 0.1, rng.int()),
                lambda: training.dropout_add(x, 0.1, rng[:1]), lambda: training.dropout_add(x, 0.1, (1, 2)),
                lambda: training.dropout_add(x, 0.1, rng, x[:2]), lambda: training.dropout_add(x, 0.1, rng, x.half()),
                lambda: training.dropout_add(x, 0.1, rng, x, torch.ones(4)),
                lambda: training.dropout_add(x, 0.1, rng, x, torch.ones(8, dtype=torch.float16)),
                lambda: training.dropout_add_backward(x.half(), x, 0.1, rng),
                lambda: training.dropout_add_backward(x[:1], x, 0.1, rng)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(ValueError, match="CUDA devices only"):
        training.dropout_add(x, 0.1, rng)


def test_attention_refuses():
    q, k = torch.zeros(2, 5, 4, 16), torch.zeros(2, 7, 2, 16)
    lens = torch.zeros(2, dtype=torch.int32)
    lse = torch.zeros(2, 4, 5)
    for bad in (lambda: training.attention(q[0], k, k), lambda: training.attention(q, k, k[:, :6]),
                lambda: training.attention(q, k.half(), k), lambda: training.attention(q[:1], k, k),
                lambda: training.attention(q[:, :, :3], k, k), lambda: training.attention(q[..., :8], k, k),
                lambda: training.attention(torch.zeros(1, 1, 1, 129), torch.zeros(1, 1, 1, 129),
                                           torch.zeros(1, 1, 1, 129)),
                lambda: training.attention(q, k[:, :, :0], k[:, :, :0]),
                lambda: training.attention(q, k, k, scale=float("inf")),
                lambda: training.attention(q, k, k, q_lens=lens.long()),
                lambda: training.attention(q, k, k, k_lens=lens[:1]),
                lambda: training.attention(q, k, k, k_lens=[1, 2]),
                lambda: training.attention(q[None], k, k),
                lambda: training.attention_backward(q[:, :4], q, k, k, q, lse),
                lambda: training.attention_backward(q, q, k, k, q.half(), lse),
                lambda: training.attention_backward(q, q, k, k, q, lse[:1])):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(ValueError, match="CUDA devices only"):
        training.attention(q, k, k, q_lens=lens, k_lens=lens)


def test_rows_of_any_layout():
    """The (outer, inner, strides) of a tensor address exactly its rows."""
    def rows(t):
        t2, outer, inner, so, si = training._rows(t)
        flat = t2.as_strided((outer, inner, t.shape[-1]), (so, si, 1), t2.storage_offset())
        return flat.reshape(t.shape), t2

    base = torch.arange(2 * 3 * 4 * 5 * 6.0).view(2, 3, 4, 5, 6)
    cases = {
        "contiguous": (base, True), "slice": (base[:, 1:], True), "one row": (base[1, 2, 3, 4], True),
        "transposed": (base.transpose(1, 2), False), "two levels": (base[:, :, :3], True),
        "expanded": (base[0, 0, 0, :1].expand(7, 6), True), "last axis strided": (base[..., ::2], False),
        "three levels": (base[:, :2, :, :4], False), "single axes": (base[:1, :1, :, :3], True),
        "one column": (base[..., :1], True),
    }
    for name, (t, in_place) in cases.items():
        got, used = rows(t)
        assert torch.equal(got, t), name
        assert (used.data_ptr() == t.data_ptr()) == in_place, name


def test_two_layouts_share_a_split():
    a = torch.arange(6 * 4 * 3.0).view(6, 4, 3)
    b = torch.arange(2 * 3 * 5 * 3.0).view(6, 5, 3)[:, :4]
    c = torch.arange(12 * 2 * 2 * 3.0).view(12, 4, 3)[::2].transpose(0, 0)
    for x, y in ((a, b), (b, a), (b, c), (a, a), (b, b)):
        x, y = x.reshape(x.shape), y
        rx, ry = training._same_split(training._rows(x), training._rows(y))
        assert rx[1:3] == ry[1:3]
        for t, r in ((x, rx), (y, ry)):
            flat = r[0].as_strided((r[1], r[2], 3), (r[3], r[4], 1), r[0].storage_offset())
            assert torch.equal(flat.reshape(t.shape), t)
    # Two-level layouts with different splits: one of them is copied.
    x = torch.arange(4 * 4 * 3.0).view(4, 4, 3)[:, :3]
    y = torch.arange(3 * 5 * 3.0).view(3, 5, 3)[:, :4]
    rx, ry = training._same_split(training._rows(x), training._rows(y))
    assert rx[1:3] == ry[1:3] and rx[1] * rx[2] == 12


def test_philox_known_answers():
    """The published known-answer vectors of Philox-4x32-10: counter and key all zeros, and all ones."""
    assert [int(w) for w in philox_words(0, 0, 0, 4)] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]


def _params(**kw):
    p = _lib.AttnTrainParams()
    base = dict(dtype=_lib.DTYPE_BF16, outer=2, inner=1, heads=4, kv_heads=2, lq=100, lk=200, hd=64, causal=0,
                scale=0.125)
    for n, v in {**base, **kw}.items():
        setattr(p, n, v)
    return p


def test_workspace_queries_check_their_arguments():
    lib = _lib.load()
    n = ctypes.c_longlong(-1)
    assert lib.unblend_attention_workspace(ctypes.byref(_params()), 1, ctypes.byref(n)) == 0 and n.value >= 4 * 800
    for bad in (dict(dtype=3), dict(outer=0), dict(kv_heads=3), dict(hd=129), dict(hd=0), dict(lq=0), dict(lk=-1),
                dict(outer=1 << 30, inner=1 << 30), dict(lq=1 << 30), dict(outer=1 << 20, heads=1 << 10, kv_heads=2)):
        assert lib.unblend_attention_workspace(ctypes.byref(_params(**bad)), 0, ctypes.byref(n)) == _lib.ERR_INVALID
    assert lib.unblend_attention_workspace(None, 0, ctypes.byref(n)) == _lib.ERR_INVALID
    assert lib.unblend_attention_workspace(ctypes.byref(_params()), 0, None) == _lib.ERR_INVALID
    assert lib.unblend_layer_norm_grad_workspace(1000, 64, ctypes.byref(n)) == 0 and n.value >= 8 * 64
    assert lib.unblend_layer_norm_grad_workspace(10, 64, ctypes.byref(n)) == 0 and n.value == 0
    assert lib.unblend_layer_norm_grad_workspace(0, 64, ctypes.byref(n)) == _lib.ERR_INVALID
    assert lib.unblend_dropout_add_grad_workspace(10, 65, ctypes.byref(n)) == 0 and n.value >= 4 * 65
    assert lib.unblend_dropout_add_grad_workspace(1 << 31, 65, ctypes.byref(n)) == _lib.ERR_INVALID


def test_entry_points_refuse_before_they_launch():
    """Null pointers, missing workspaces and unknown types return an error code; nothing here reaches a GPU."""
    lib = _lib.load()
    x = ctypes.create_string_buffer(64)
    p = ctypes.addressof(x)
    bad = _lib.ERR_INVALID
    assert lib.unblend_layer_norm_forward(None, 0, 4, p, p, p, p, 1e-5, 1, 1, 4, 0, 0, None) == bad
    assert lib.unblend_layer_norm_forward(p, 0, 4, p, p, p, p, -1.0, 1, 1, 4, 0, 0, None) == bad
    assert lib.unblend_layer_norm_forward(p, 0, 4, p, p, p, p, 1e-5, 1, 1, 4, 0, 1, None) == bad
    assert lib.unblend_layer_norm_forward(p, 0, 4, p, p, p, p, 1e-5, 1 << 20, 1 << 20, 4, 0, 0, None) == bad
    assert lib.unblend_layer_norm_backward(p, 0, 4, p, 0, 4, p, p, p, p, None, p, 1, 1, 4, 0, 0, None) == bad
    assert lib.unblend_layer_norm_backward(p, 0, 4, p, 0, 4, p, p, p, p, p, None, 1, 1000, 4, 0, 0, None) == bad
    assert lib.unblend_dropout_add_forward(p, 0, 4, p, 0, 4, p, p, 1.5, p, 1, 1, 4, 0, 0, 0, None) == bad
    assert lib.unblend_dropout_add_forward(p, 0, 4, p, 0, 4, p, p, 0.5, p + 4, 1, 1, 4, 0, 0, 0, None) == bad
    assert lib.unblend_dropout_add_forward(p, 0, 4, p, 0, 4, p, p, 0.5, p, 1, 1, 4, 0, 1, 0, None) == bad
    assert lib.unblend_dropout_add_backward(p, 0, 4, p, 0, 4, None, p, p, p, 0.5, p, 1, 1, 4, 0, 0, 0, None) == bad
    a = _params()
    assert lib.unblend_attention_forward(p, p, None, p, p, None, 0, ctypes.byref(a), None) == bad
    assert lib.unblend_attention_forward(p, p, p, p, p, None, 0, ctypes.byref(_params(heads=5)), None) == bad
    assert lib.unblend_attention_backward(p, p, p, p, p, p, p, p, p, None, 0, ctypes.byref(a), None) == bad
    assert lib.unblend_attention_backward(p, p, p, p, p, p, p, p, p, p & ~15, 16, ctypes.byref(a), None) == bad


@pytest.mark.parametrize("ctype,cname", [(_lib.HeadStrides, "UnblendHeadStrides"),
                                         (_lib.AttnTrainParams, "UnblendAttnTrainParams")])
def test_param_struct_layout(tmp_path, ctype, cname):
    from test_capi import test_param_struct_layout_matches_c

    test_param_struct_layout_matches_c(tmp_path, ctype, cname)
