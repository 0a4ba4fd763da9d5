"""Rotary operators on the GPU: layouts and values at the edge of what they take, against their 64-bit definitions."""

from __future__ import annotations

import pytest
import torch

from test_rotary_gpu import BF16, F16, F32, _check_norm, _check_rotary, _rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("interleaved", [True, False])
def test_one_head_of_any_stride(interleaved, t):
    """A single head is never stepped over: its stride may be off every boundary, with rows on them. One head on both
    sides, beside many (which divide a token among teams) and beside none, whole rows and rows by way of shared memory."""
    pad = 4 if t != F32 else 2  # two heads and their padding are whole 16-byte pieces, one head is not
    for hd, pairs in ((64, 32), (64, 6), (64, 25), (32, 16), (128, 64)):
        f, w = _rand(pairs, seed=1), _rand(hd, seed=2, shift=1.0)
        for batch, length in ((1, 1), (3, 20), (2, 3001)):
            one = _rand(batch, length, 2, hd + pad, seed=3, t=t)[..., :1, :hd]
            other = _rand(batch, length, 2, hd + pad, seed=4, t=t)[..., :1, :hd]
            assert one.stride(-2) * one.element_size() % 16 and one.stride(-3) * one.element_size() % 16 == 0
            many = _rand(batch, length, 16, hd, seed=5, t=t)
            for q, k in ((one, None), (one, other), (many, one), (one, many)):
                dk = None if k is None else other if k.shape[-2] == 1 else many
                _check_rotary(q, k, f, None, interleaved)
                _check_norm(q, k, w, None if k is None else w, f, None, interleaved,
                            dq=other if q.shape[-2] == 1 else many, dk=dk)
