"""Calls of the training operators at the edge of what they allow: alignment, sizes, workspaces, refusals. No GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

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
