"""Rotary operators on the GPU: layouts and values at the edge of what they take, against their 64-bit definitions."""

from __future__ import annotations

import math

import pytest
import torch

from rotary_reference import TURN16
from test_rotary_gpu import BF16, F16, F32, _check_norm, _check_rotary, _rand
from training_reference import assert_within, half
from unblend_b200 import training

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


@pytest.mark.parametrize("outer,inner,length,heads", [(3, 7, 999983, 1), (1, 1, 20000003, 1), (4194301, 5, 1, 1),
                                                      (2, 4194305, 2, 1), (1, 3, 5, 1 << 20), (1, 1, 2, 999979),
                                                      (32768, 1, 512, 1), (1, 65536, 255, 1)])
def test_every_row_is_found(outer, inner, length, heads):
    """Axes of many sizes around powers of two and primes: each row turns by the position given for it, an angle that is
    its number. x = 1 + 0 i becomes its cosine and sine."""
    x = torch.zeros(outer, inner, length, heads, 2, device="cuda", dtype=BF16)
    x[..., 0] = 1
    rows = outer * inner * length
    number = torch.arange(rows, device="cuda").view(outer, inner, length)
    f = torch.ones(1, device="cuda", dtype=torch.float64)
    y = training.rotary_forward(x, None, f, number)[0].view(rows, heads, 2)
    for first in range(0, rows, 1 << 21):  # not all in 64 bits at a time
        part = slice(first, first + (1 << 21))
        a = number.view(-1)[part, None].double()
        want = torch.stack((a.cos(), a.sin()), -1)
        assert_within("turned", y[part], want.expand(-1, heads, -1), half(BF16) * want.abs() + TURN16 + 2.0**-133)
    y = training.rotary_forward(x, None, f)[0].view(-1, length, heads, 2)
    assert torch.equal(y[:1].expand_as(y), y)  # rows counted from 0 in each sequence


@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("interleaved", [True, False])
def test_norm_keeps_infinities_behind_the_pairs(interleaved, t):
    """An infinity behind the pairs makes its row's reciprocal root 0: it becomes NaN itself, the other dims 0. Infinite and
    NaN weights there reach no other dim either."""
    for hd, pairs in ((64, 5), (64, 8), (64, 0), (50, 7), (128, 32), (33, 16)):
        f, w = _rand(pairs, seed=1), _rand(hd, seed=2, shift=1.0)
        for at in range(2 * pairs, hd, 3):
            x = _rand(2, 9, 3, hd, seed=3, t=t)
            clean = training.qk_norm_rotary_forward(x, None, w, None, f, None, interleaved)[0]
            x[1, 4, 2, at], x[0, 8, 0, at] = math.inf, -math.inf
            y = training.qk_norm_rotary_forward(x, None, w, None, f, None, interleaved)[0]
            want = clean.clone()
            for row in ((1, 4, 2), (0, 8, 0)):
                want[row] = 0
                want[(*row, at)] = math.nan
            assert torch.equal(y.nan_to_num(7.0), want.nan_to_num(7.0)), (hd, pairs, at)
            x = _rand(2, 9, 3, hd, seed=3, t=t)
            for bad in (math.inf, math.nan):
                g = w.clone()
                g[at] = bad
                y = training.qk_norm_rotary_forward(x, None, g, None, f, None, interleaved)[0]
                assert not y[..., at].isfinite().any()
                y[..., at] = clean[..., at]
                assert torch.equal(y, clean), (hd, pairs, at)


@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("interleaved", [True, False])
def test_bits_behind_the_pairs(interleaved, t):
    """What does not turn comes through bit for bit, signs of zeros and subnormal numbers too; NaN stay NaN."""
    whole = torch.int32 if t == F32 else torch.int16
    tiny, most = torch.finfo(t).smallest_normal, torch.finfo(t).max
    values = torch.tensor([-0.0, math.inf, 0.0, -math.inf, math.nan, tiny / 4, -tiny / 2, most, -most, 1.0], device="cuda")
    for hd, pairs in ((64, 5), (64, 8), (64, 0), (50, 7), (128, 32), (33, 16), (256, 100)):
        f = _rand(pairs, seed=1)
        q = _rand(2, 9, 3, hd, seed=2, t=t)
        behind = q[..., 2 * pairs:]
        behind.copy_(values.to(t).repeat(behind.numel() // 10 + 1)[:behind.numel()].view(behind.shape))
        for call in (training.rotary_forward, training.rotary_backward):
            y = call(q, None, f, None, interleaved, 3.0)[0]
            got, nan = y[..., 2 * pairs:], behind.isnan()
            assert nan.any() and torch.equal(got.isnan(), nan)
            assert torch.equal(got.contiguous().view(whole)[~nan], behind.contiguous().view(whole)[~nan]), (hd, pairs)
            assert y[..., :2 * pairs].isfinite().all()
