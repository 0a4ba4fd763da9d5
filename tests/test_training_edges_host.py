"""Calls of the training operators at the edge of what they allow: alignment, sizes, workspaces, refusals. No GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

from training_reference import philox_words
from unblend_b200 import _lib, training


def _buffer(n: int = 256) -> tuple[ctypes.Array, int]:
    """A host buffer (kept by the caller) and a 16-byte aligned address in it."""
    x = ctypes.create_string_buffer(n + 16)
    return x, (ctypes.addressof(x) + 15) & ~15


def test_row_statistics_need_their_alignment():
    """(mean, rstd) are moved as one 8-byte access: an address off that boundary must be refused, not launched."""
    lib = _lib.load()
    keep, p = _buffer()
    bad = _lib.ERR_INVALID
    assert lib.unblend_layer_norm_forward(p, 0, 4, p, p + 4, p, p, 1e-5, 1, 1, 4, 0, 0, None) == bad
    assert lib.unblend_layer_norm_backward(p, 0, 4, p, 0, 4, p + 4, p, p, None, None, None, 1, 1, 4, 0, 0, None) == bad


def test_statistics_off_their_alignment_are_copied(monkeypatch):
    """``stats`` in the middle of a larger buffer: contiguous, but on a 4-byte boundary."""
    seen = {}
    monkeypatch.setattr(training, "_check_cuda", lambda *a: None)
    monkeypatch.setattr(training, "_launch", lambda t, name, *args, **kw: seen.update({name: args}))
    buf = torch.zeros(33)
    at = next(o for o in (0, 1) if (buf.data_ptr() + 4 * o) % 8)
    stats = buf[at:at + 32].view(16, 2)
    assert stats.is_contiguous() and stats.data_ptr() % 8
    x = torch.zeros(16, 8)
    training.layer_norm_backward(x, x, stats)
    assert seen["unblend_layer_norm_backward"][6] % 8 == 0


def _attention_workspace(backward=False, **kw):
    p = _lib.AttnTrainParams()
    base = dict(dtype=_lib.DTYPE_BF16, outer=1, inner=1, heads=8, kv_heads=8, lq=100, lk=100, hd=64, causal=0,
                scale=0.125)
    for name, v in {**base, **kw}.items():
        setattr(p, name, v)
    n = ctypes.c_longlong(-1)
    assert _lib.load().unblend_attention_workspace(ctypes.byref(p), int(backward), ctypes.byref(n)) == 0
    return n.value


@pytest.mark.parametrize("dtype", [_lib.DTYPE_F32, _lib.DTYPE_BF16, _lib.DTYPE_F16])
@pytest.mark.parametrize("kw", [
    dict(lq=8192, lk=8192, heads=16, kv_heads=4, hd=128, causal=1), dict(outer=8, lq=2688, lk=1344),
    dict(inner=62, lq=801, lk=801), dict(lq=65536, lk=65536, heads=32, kv_heads=8, hd=128),
    dict(inner=801, lq=62, lk=62), dict(outer=64, lq=300, lk=8000, heads=16, kv_heads=1)])
def test_calls_that_fill_the_gpu_need_no_forward_workspace(kw, dtype):
    """Parts of split keys are for calls with too few rows of queries: no room for them where there are enough."""
    assert _attention_workspace(dtype=dtype, **kw) == 0


def test_workspace_is_what_the_parts_take():
    """A few rows per key/value head are split into at most 32 parts, other calls into what four waves of CTAs take."""
    # 4 sequences of 4 key/value heads: 592 CTAs wanted, 32 parts each of 64 rows with their sums.
    assert _attention_workspace(outer=4, lq=1, lk=8191, heads=16, kv_heads=4, hd=128) == 32 * 64 * 129 * 4
    for dtype in (_lib.DTYPE_F32, _lib.DTYPE_BF16, _lib.DTYPE_F16):
        size = 4 if dtype == _lib.DTYPE_F32 else 2
        for outer, heads, kv, lq, lk, hd in ((1, 8, 8, 300, 5000, 64), (2, 16, 4, 40, 4097, 128),
                                             (1, 1, 1, 17, 9000, 40), (3, 4, 2, 129, 700, 96), (1, 2, 2, 8, 100000, 64),
                                             (7, 8, 1, 2, 3000, 72),
                                             (1, 4, 4, 5000, 130, 64), (1, 1, 1, 1, 1, 1)):
            few = heads // kv * lq <= (8 if size == 4 else 16) and hd * size % 16 == 0
            tiles = outer * heads * -(-lq // 64)
            parts = max(1, 4 * 296 // tiles, 32 if few else 1)
            if tiles >= 296 and not few:
                parts = 0
            rows = outer * heads * lq
            kw = dict(dtype=dtype, outer=outer, heads=heads, kv_heads=kv, lq=lq, lk=lk, hd=hd)
            assert _attention_workspace(**kw) <= 4 * min(32, parts) * rows * (hd + 1)
            key_rows, key_tiles = outer * kv * lk, outer * kv * -(-lk // 64)
            most = 4 * (3 * rows + 8 + 4 * outer * kv)  # statistics, norms, ranges
            most += 4 * min(32, max(0 if tiles >= 296 else 1, 4 * 296 // tiles)) * rows * hd
            most += 8 * min(32, max(0 if key_tiles >= 296 else 1, 4 * 296 // key_tiles)) * key_rows * hd
            assert _attention_workspace(True, **kw) <= most + 64


def test_forward_mode_derivatives_are_refused(monkeypatch):
    """A dual tensor has ``requires_grad`` false: it must not pass as a plain one, its tangent lost without a word."""
    import torch.autograd.forward_ad as fwd

    monkeypatch.setattr(training, "_check_cuda", lambda *a: None)
    monkeypatch.setattr(training, "_launch", lambda *a, **kw: None)
    x, w, q = torch.randn(3, 8), torch.ones(8), torch.randn(1, 3, 2, 8)
    rng = torch.zeros(2, dtype=torch.int64)
    with fwd.dual_level():
        dx, dw, dq = (fwd.make_dual(t, torch.ones_like(t)) for t in (x, w, q))
        for call in (lambda: training.layer_norm(dx), lambda: training.layer_norm(x, dw),
                     lambda: training.layer_norm(x, w, dw), lambda: training.attention(dq, q, q),
                     lambda: training.attention(q, dq, q), lambda: training.attention(q, q, dq),
                     lambda: training.dropout_add(dx, 0.1, rng), lambda: training.dropout_add(x, 0.1, rng, dx),
                     lambda: training.dropout_add(x, 0.1, rng, x, dw)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call()
        training.layer_norm(x, w)  # no tangents: a plain call, inside a dual level too


def test_sizes_beyond_the_kernels_are_value_errors(monkeypatch):
    """As every wrong argument, and before anything is allocated or launched. Expanded tensors need no memory here."""
    monkeypatch.setattr(training, "_launch", lambda *a, **kw: pytest.fail("launched"))
    rng = torch.zeros(2, dtype=torch.int64)
    for shape in ((1 << 31, 1), (1 << 16, 1 << 16, 1), (1, 1 << 31)):
        x = torch.zeros((1,) * len(shape)).expand(shape)
        rows = x.numel() // shape[-1]
        for call in (lambda: training.layer_norm_forward(x),
                     lambda: training.layer_norm_backward(x, x, torch.zeros(1, 1).expand(rows, 2)),
                     lambda: training.dropout_add_forward(x, 0.5, rng),
                     lambda: training.dropout_add_backward(x, x, 0.5, rng)):
            with pytest.raises(ValueError, match="rows"):
                call()
    for shape in ((1, 1 << 30, 1, 1), (1 << 31, 1, 1, 1), (1 << 16, 1 << 16, 1, 1, 1), (1, (1 << 32) + 5, 1, 1),
                  (1 << 20, 1, 1 << 10, 1), (1, 1, 1 << 32, 1)):
        q = torch.zeros((1,) * len(shape)).expand(shape)
        lse = torch.zeros(1, 1, 1).expand(q.numel() // shape[-3] // shape[-2], shape[-2], shape[-3])
        with pytest.raises(ValueError, match="beyond"):
            training.attention_forward(q, q, q)
        with pytest.raises(ValueError, match="beyond"):
            training.attention_backward(q, q, q, q, q, lse)


def test_arguments_that_fp32_cannot_hold_and_missing_results():
    q, x = torch.zeros(1, 2, 1, 8), torch.zeros(2, 8)
    for call in (lambda: training.attention(q, q, q, scale=1e39), lambda: training.attention(q, q, q, scale=-1e300),
                 lambda: training.layer_norm_backward(x, x, None), lambda: training.layer_norm_backward(x, x, 1.0),
                 lambda: training.attention_backward(q, q, q, q, q, None)):
        with pytest.raises(ValueError) as e:
            call()
        assert "CUDA devices only" not in str(e.value)


def test_dropout_keeps_its_input_only_for_the_scale(monkeypatch):
    """The branch's activations are read for the LayerScale's gradient alone; without it they may be freed."""
    launched = []
    monkeypatch.setattr(training, "_check_cuda", lambda *a: None)
    monkeypatch.setattr(training, "_refuse_capture", lambda *a: None)
    monkeypatch.setattr(training, "_launch", lambda t, name, *args, **kw: launched.append((name, args)))
    rng, w = torch.zeros(2, dtype=torch.int64), torch.ones(8)
    for x_dtype in (torch.float32, torch.bfloat16):
        for scale in (None, w, w.clone().requires_grad_()):
            x = torch.randn(5, 3, 8, dtype=x_dtype).requires_grad_()
            res = torch.randn(5, 3, 8)
            y = training.dropout_add(x, 0.1, rng, res, scale)
            kept = [t.data_ptr() for t in y.grad_fn.saved_tensors if t is not None]
            learns = scale is not None and scale.requires_grad
            assert (x.data_ptr() in kept) == learns
            y.backward(torch.ones(5, 3, 8))
            assert x.grad.shape == x.shape and x.grad.dtype == x_dtype
            name, args = launched[-1]
            assert name == "unblend_dropout_add_backward" and (args[3] == x.data_ptr()) == learns
            assert not learns or scale.grad.shape == w.shape
            assert args[12:15] == (1, 15, 8) and args[15:17] == (training._DTYPES[x_dtype], _lib.DTYPE_F32)


def test_launch_counts_are_what_a_call_launches(monkeypatch):
    """Layer norm's backward pass is one kernel, two where partial sums are joined, three for rows over 8192 columns;
    dropout's two with a scale's gradient."""
    counts = []
    monkeypatch.setattr(training, "_check_cuda", lambda *a: None)
    monkeypatch.setattr(training, "_launch", lambda t, name, *args, kernels=1: counts.append(kernels))
    for rows, cols, weights, want in ((64, 512, True, 1), (65, 512, True, 2), (1000, 512, False, 1), (1, 1024, True, 1),
                                      (1, 1025, True, 1), (2, 1025, True, 2), (2, 8192, False, 1), (1, 8193, True, 3),
                                      (300, 9000, True, 3), (300, 9000, False, 1)):
        x = torch.zeros(rows, cols)
        training.layer_norm_backward(x, x, torch.zeros(rows, 2), weight_grads=weights)
        assert counts.pop() == want, (rows, cols, weights)
    x, rng, w = torch.zeros(4, 8), torch.zeros(2, dtype=torch.int64), torch.ones(8)
    for scale, grad, want in ((None, True, 1), (w, False, 1), (w, True, 2)):
        training.dropout_add_backward(x, x, 0.5, rng, scale, grad)
        assert counts.pop() == want
    training.dropout_add_forward(x, 0.5, rng)
    training.layer_norm_forward(x)
    assert counts == [1, 1]


def test_philox_against_all_published_vectors():
    """Philox-4x32-10 by the paper's definition in Python integers, against its three known answers, and the words that
    the other tests use against that."""
    def philox(counter, key):
        c, k = list(counter), list(key)
        for _ in range(10):
            a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
            c = [(b >> 32) ^ c[1] ^ k[0], b & 0xFFFFFFFF, (a >> 32) ^ c[3] ^ k[1], a & 0xFFFFFFFF]
            k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
        return c

    ones = 0xFFFFFFFF
    assert philox([0] * 4, [0] * 2) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert philox([ones] * 4, [ones] * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert philox([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], [0xA4093822, 0x299F31D0]) == \
        [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]
    for seed, offset, block in ((-1, -1, 0), (1 << 62, 3, 5), (-(1 << 63), 1 << 40, (1 << 60) + 7), (77, -2, 1 << 33)):
        want = philox([block & ones, block >> 32, offset & ones, (offset >> 32) & ones],
                      [seed & ones, (seed >> 32) & ones])
        assert [int(w) for w in philox_words(seed, offset, 4 * block, 4)] == want


def test_lazily_negated_views_are_refused(monkeypatch):
    """``z.conj().imag`` shares z's memory with a sign that only torch's own operators apply."""
    monkeypatch.setattr(training, "_check_cuda", lambda *a: None)
    monkeypatch.setattr(training, "_launch", lambda *a, **kw: pytest.fail("launched"))
    x = torch.randn(4, 8, dtype=torch.complex64).conj().imag
    assert x.is_neg()
    q, plain, rng = x.view(1, 4, 1, 8), torch.zeros(4, 8), torch.zeros(2, dtype=torch.int64)
    for call in (lambda: training.layer_norm(x), lambda: training.layer_norm_backward(x, plain, torch.zeros(4, 2)),
                 lambda: training.attention(q, q, q), lambda: training.dropout_add(plain, 0.1, rng, x),
                 lambda: training.dropout_add(plain, 0.1, rng, None, x[0]),
                 lambda: training.dropout_add_backward(x, plain, 0.1, rng)):
        with pytest.raises(ValueError, match="resolve_neg"):
            call()
    torch.testing.assert_close(x.resolve_neg(), x)
