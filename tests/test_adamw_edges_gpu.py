"""AdamW and the norm of gradients on the GPU at the edge of what they take."""

from __future__ import annotations

import pytest
import torch

from adamw_reference import M_TABLE, U_TABLE, codes
from test_adamw_gpu import BF16, F32, _check_step, _gen, _model, _state
from unblend_b200 import training

pytestmark = pytest.mark.gpu


def test_every_ratio_gets_its_code():
    """All fp32 numbers of 18 octaves as moments relative to a largest of 1, above, between and below the codes. With beta =
    0 the step takes m = g, and u = sqrt(g^2) = g: the root of a rounded square is the number again in radix 2."""
    n = 1 << 23
    p = [torch.zeros((n + 254) // 255 * 256, device="cuda")]
    state = training.adamw_state(p, 8)
    for octave in range(18):
        w = torch.arange(n, device="cuda", dtype=torch.int32) + ((127 - 1 - octave) << 23)
        g = w.view(F32)
        g = torch.nn.functional.pad(torch.where(w % 3 == 0, -g, g), (0, -n % 255)).view(-1, 255)
        g = torch.nn.functional.pad(g, (1, 0), value=1.0).view(-1)
        training.adamw_step(p, [g], state, 2, betas=(0.0, 0.0), eps=1.0)
        assert bool((state.scales == 1).all())
        m, _ = codes(g, M_TABLE)
        same = (m == state.exp_avg) | ((m & 127 == 0) & (state.exp_avg & 127 == 0))
        assert bool(same.all()), octave
        u, _ = codes(g.abs(), U_TABLE)
        assert torch.equal(u, state.exp_avg_sq), octave


def test_roots_are_rounded_correctly():
    """The scales of u are the roots of v, rounded once, for any size of v; zeros and NaN among them. One element
    of each block has a moment, no gradient."""
    n = 1 << 17
    s = torch.exp2(torch.rand(n, device="cuda", generator=_gen(1)) * 136 - 73)  # s^2 from 2^-146 to 2^126
    s[:4] = torch.tensor([0.0, 1.8e19, float("nan"), 1e-30], device="cuda")
    p = [torch.zeros(n * 256, device="cuda")]
    state = training.adamw_state(p, 8)
    state.exp_avg_sq[77::256] = 255
    state.scales[:, 1] = s
    v = (s * s) * torch.tensor(0.9, dtype=F32, device="cuda")
    training.adamw_step(p, [torch.zeros_like(p[0])], state, 2, betas=(0.5, 0.9))
    want = v.double().sqrt().float()  # 53 bits are enough for the second rounding to change nothing
    assert want[1].isfinite() and int(want.isnan().sum()) == 1
    assert torch.equal(state.scales[:, 1].nan_to_num(-1.0), want.nan_to_num(-1.0))
    assert not state.scales[:, 0].any()


@pytest.mark.parametrize("n", [1000, 3_000_000])  # one kernel, partial sums and a join
def test_a_norm_beyond_fp32_skips_the_step(n):
    """Finite gradients whose norm is no fp32 number: infinite, as it is handed out, and its factor NaN."""
    grads = [torch.full((n,), 3e38, device="cuda")]
    norm, scale = training.grad_norm(grads, 1.0)
    assert norm.isinf() and scale.isnan()
    p = [torch.ones(n, device="cuda")]
    for bits in (32, 8):
        state = training.adamw_state(p, bits)
        training.adamw_step(p, grads, state, 1, grad_scale=scale)
        assert bool((p[0] == 1).all()) and not any(bool(x.any()) for x in state if x is not None)
    largest = torch.finfo(F32).max
    norm, scale = training.grad_norm([torch.tensor([largest], device="cuda")], 1.0)  # the last one that is
    assert float(norm) == largest and float(scale) == pytest.approx(1 / largest, rel=0, abs=2.0**-149)


@pytest.mark.parametrize("bits", [32, 8])
def test_neighbours_in_one_buffer(bits):
    """Parameters, gradients, moments, scales and the numbers of a step side by side in one allocation are apart."""
    params, grads = _model(1, BF16)
    state = _state(params, bits, 2)
    parts = [*params, *grads, *(x for x in state if x is not None)]
    size = [-(-x.nbytes // 16) * 16 for x in parts]
    raw = torch.zeros(sum(size) + 32, device="cuda", dtype=torch.uint8)
    inside = [x[:y.nbytes].view(y.dtype).view(y.shape) for x, y in zip(raw.split([*size, 32])[:-1], parts)]
    for x, y in zip(inside, parts):
        x.copy_(y)
    n = len(params)
    number, lr, gs = raw[-32:-24].view(torch.int64), raw[-24:-20].view(F32), raw[-16:-12].view(F32)
    number.fill_(7), lr.fill_(1e-3), gs.fill_(0.5)
    for p, g, s in ((params, grads, state), (inside[:n], inside[n:2 * n], training.AdamWState(*inside[2 * n:]))):
        training.adamw_step(p, g, s, number, lr, grad_scale=gs)
    for x, y in zip(inside, parts):
        assert torch.equal(x, y)
    assert int(number) == 7 and float(gs) == 0.5


@pytest.mark.parametrize("bits", [32, 8])
def test_many_steps(bits):
    """Each of 150 steps from the state that the one before left, gradients of changing sizes."""
    sizes = [(300,), (64, 5), (7,)]
    params, grads = _model(3, BF16, sizes=sizes)
    state = training.adamw_state(params, bits)
    for n in range(1, 151):
        for i, g in enumerate(grads):
            g.copy_(torch.randn(g.shape, device="cuda", generator=_gen(10 * n + i)) * 10.0 ** (i - 3 - n // 50))
        _check_step(params, grads, state, n, betas=(0.9, 0.999))


def test_second_moments_in_8_bits_beside_a_larger_one():
    """A root that shrinks by 0.05 % per step beside a steady one stays where it is, one that shrinks by 5 % (more than
    half a code, at most 1/32) moves on with each step, and a block that shrinks as a whole does so by its scale."""
    p, zero = [torch.zeros(256, device="cuda")], torch.zeros(256, device="cuda")
    steady = zero.clone()
    steady[0] = 1.0
    for beta2, grad, steps in ((0.999, steady, 400), (0.999, zero, 400), (0.9, steady, 50)):
        state = training.adamw_state(p, 8)
        state.exp_avg_sq.copy_(torch.arange(255, -1, -1, device="cuda").clamp(min=100))
        state.scales[:, 1] = 1.0
        before = state.exp_avg_sq.clone()
        for n in range(steps):
            training.adamw_step(p, [grad], state, n + 1, betas=(0.9, beta2))
        if beta2 == 0.9:
            assert state.exp_avg_sq[0] == 255
            assert bool((before[1:].int() - state.exp_avg_sq[1:].int() >= steps).all())
        else:
            assert torch.equal(state.exp_avg_sq, before)
        # each step rounds its products and the root: 4 U
        want = 1.0 if grad is steady else 0.999 ** (steps / 2)
        assert abs(float(state.scales[0, 1]) - want) <= steps * 4 * 2.0**-24 * want + 3e-8 * steps * (grad is steady)


def test_moments_behind_2_to_31():
    """The last elements of a large tensor, over two steps, are those of a small one bit for bit; nothing else changes."""
    n = (1 << 31) + 1001
    start = (n - 3000) // 256 * 256
    p, g = torch.zeros(n, device="cuda", dtype=BF16), torch.zeros(n, device="cuda", dtype=BF16)
    small = [(torch.randn(n - start, device="cuda", generator=_gen(s)) * 0.1).to(BF16) for s in (1, 2)]
    p[start:], g[start:] = small
    state, little = training.adamw_state([p], 8), training.adamw_state(small[:1], 8)
    for step in (1, 2):
        training.adamw_step([p], [g], state, step)
        _check_step(small[:1], small[1:], little, step, 1.0, lr=1e-3, betas=(0.9, 0.999), weight_decay=0.01)
        for big, x, at in ((p, small[0], start), (state.exp_avg, little.exp_avg, start),
                           (state.exp_avg_sq, little.exp_avg_sq, start), (state.scales, little.scales, start // 256)):
            assert torch.equal(big[at:], x) and bool(x.any())
            assert not big[:at].any()
