"""Wrong kinds of arguments of the rotary operators and the gradient norm. No GPU needed."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from unblend_b200 import training

F = torch.ones(8)
Q, K = torch.zeros(2, 5, 4, 16), torch.zeros(2, 5, 2, 16)


@pytest.mark.parametrize("call", [training.rotary, training.rotary_forward, training.rotary_backward,
                                  lambda q, k, f, pos=None, **kw: training.qk_norm_rotary(q, k, None, None, f, pos, **kw)])
def test_kinds_of_arguments(call):
    pos = torch.arange(5)
    for scale in ("1", None, [1.0], 1j, 10**400, torch.ones(2), torch.ones(0)):
        with pytest.raises(ValueError, match="scale"):
            call(Q, K, F, scale=scale)
    for scale in (1, 0.5, True, np.float32(0.5), torch.tensor(0.5), torch.ones(1)):  # what Python takes for a number
        with pytest.raises(ValueError, match="CUDA devices only"):
            call(Q, K, F, scale=scale)
    with pytest.raises(ValueError, match="freqs"):
        call(Q, K, F.to_sparse())
    with pytest.raises(ValueError, match="positions"):
        call(Q, K, F, pos.to_sparse())


def test_sparse_lengths():
    with pytest.raises(ValueError, match="lens"):
        training.qk_norm_rotary(Q, K, None, None, F, lens=torch.ones(2, dtype=torch.int32).to_sparse())


def test_frequencies_refuse_what_is_no_number():
    for bad in (dict(base="10"), dict(base=None), dict(base=10**400), dict(factor="2"), dict(factor=None), dict(factor=[2.0]),
                dict(method="parts", trained_length=9, slow="1"), dict(method="parts", trained_length=9, fast=None),
                dict(method="parts", trained_length=9, slow=math.nan), dict(method=None)):
        with pytest.raises(ValueError):
            training.rotary_freqs(4, **bad)
    same = training.rotary_freqs(4, 100.0, 2.0)
    assert torch.equal(training.rotary_freqs(4, np.float32(100), torch.tensor(2.0)), same)
    f = training.rotary_freqs(4, factor=2.0, method="parts", trained_length=9, fast=math.inf)
    assert torch.equal(f, training.rotary_freqs(4, factor=2.0))  # nothing turns fast enough to be kept
