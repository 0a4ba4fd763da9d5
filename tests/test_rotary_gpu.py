"""Rotary positions and the norm of queries and keys on the GPU against their 64-bit definitions."""

from __future__ import annotations

import math

import pytest
import torch

from rotary_reference import TURN, exact_angle, qk_norm_reference, rotary_reference
from training_reference import assert_within, half
from unblend_b200 import _lib, training

pytestmark = pytest.mark.gpu

F32, BF16, F16, F64 = torch.float32, torch.bfloat16, torch.float16, torch.float64


def _rand(*shape, seed, t=F32, scale=1.0, shift=0.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * scale + shift).to(t)


def _check_rotary(q, k, freqs, positions=None, interleaved=True, scale=1.0, dq=None, dk=None):
    got = training.rotary_forward(q, k, freqs, positions, interleaved, scale)
    back = training.rotary_backward(q if dq is None else dq, k if dk is None else dk, freqs, positions, interleaved,
                                    scale)
    for name, x, y, inverse in (("q", q, got[0], False), ("k", k, got[1], False),
                                ("dq", q if dq is None else dq, back[0], True),
                                ("dk", k if dk is None else dk, back[1], True)):
        if x is None:
            assert y is None
            continue
        assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
        assert_within(name, y, *rotary_reference(x, freqs, positions, interleaved, scale, inverse))
        rest = 2 * freqs.shape[0]
        assert torch.equal(y[..., rest:].nan_to_num(3.0), x[..., rest:].nan_to_num(3.0))
    again = training.rotary_forward(q, k, freqs, positions, interleaved, scale)
    assert all(a is b or torch.equal(a.nan_to_num(3.0), b.nan_to_num(3.0)) for a, b in zip(got, again))
    return got


def _check_norm(q, k, gq, gk, freqs, positions=None, interleaved=True, scale=1.0, eps=1e-6, lens=None, dq=None,
                dk=None):
    args = (gq, gk, freqs, positions, interleaved, scale, eps, lens)
    dq = _rand(*q.shape, seed=91, t=q.dtype) if dq is None else dq
    dk = None if k is None else _rand(*k.shape, seed=92, t=q.dtype) if dk is None else dk
    out = training.qk_norm_rotary_forward(q, k, *args)
    back = training.qk_norm_rotary_backward(dq, dk, q, k, *args)
    for i, (name, x, d, g) in enumerate((("q", q, dq, gq), ("k", k, dk, gk))):
        if x is None:
            assert out[i] is None and back[i] is None and back[2 + i] is None
            continue
        assert out[i].dtype == back[i].dtype == x.dtype and out[i].is_contiguous() and back[i].is_contiguous()
        ref = qk_norm_reference(x, d, g, freqs, positions, interleaved, scale, eps, lens)
        assert_within(name, out[i], *ref["y"])
        assert_within("d" + name, back[i], *ref["dx"])
        if g is None:
            assert back[2 + i] is None
        else:
            assert back[2 + i].dtype == g.dtype
            assert_within("dgamma_" + name, back[2 + i], *ref["dgamma"])
    again = training.qk_norm_rotary_backward(dq, dk, q, k, *args)
    assert all(a is b or torch.equal(a, b) for a, b in zip(back, again))
    return out, back


# (head_dim, pairs): whole heads, parts, no pair at all, pairs that end inside a chunk of eight, odd widths.
DIMS = [(64, 32), (64, 16), (64, 5), (64, 0), (8, 4), (16, 8), (40, 20), (48, 18), (96, 24), (128, 64), (128, 32),
        (160, 80), (256, 128), (256, 8), (1, 0), (2, 1), (7, 2), (33, 16), (50, 25), (100, 50), (250, 125), (255, 16)]


@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("interleaved", [True, False])
def test_rotary_dims(interleaved, t):
    for hd, pairs in DIMS:
        f = _rand(pairs, seed=hd, scale=0.7)
        q, k = _rand(2, 37, 4, hd, seed=1, t=t), _rand(2, 37, 2, hd, seed=2, t=t)
        _check_rotary(q, k, f, None, interleaved, 1.25)
        _check_rotary(q[:1, :1], None, f.double(), None, interleaved)


@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("interleaved", [True, False])
def test_norm_dims(interleaved, t):
    for hd, pairs in DIMS:
        f = _rand(pairs, seed=hd, scale=0.7)
        q, k = _rand(2, 37, 4, hd, seed=1, t=t, scale=2.0), _rand(2, 37, 2, hd, seed=2, t=t)
        gq, gk = (_rand(hd, seed=s, t=t, scale=0.3, shift=1.0) for s in (3, 4))
        _check_norm(q, k, gq, gk, f, None, interleaved, 1.25)
        _check_norm(q[:1, :1], None, gq.float(), None, f.double(), None, interleaved)


@pytest.mark.parametrize("t", [F32, BF16])
def test_lengths(t):
    """One token to thousands, with any number of teams per token."""
    f = training.rotary_freqs(64, device="cuda")
    for batch, length, h, hk in ((1, 1, 1, 1), (1, 1, 32, 1), (1, 2, 3, 5), (3, 1, 8, 8), (1, 129, 1, 1),
                                 (2, 5003, 3, 1), (700, 3, 2, 2), (1, 20011, 8, 2), (1, 4, 301, 7)):
        q, k = _rand(batch, length, h, 64, seed=5, t=t), _rand(batch, length, hk, 64, seed=6, t=t)
        _check_rotary(q, k, f)
        _check_norm(q, k, _rand(64, seed=7), _rand(64, seed=8), f, None, False)


@pytest.mark.parametrize("t", [F32, F16])
@pytest.mark.parametrize("hd", [64, 50])
def test_strides(hd, t):
    """Slices of a packed projection, token axes in another order, heads before tokens, rows off 16-byte boundaries,
    heads and rows that share memory, gradients that are expanded scalars."""
    f = _rand(hd // 2 - 1, seed=1, scale=0.5)
    gq, gk = _rand(hd, seed=2, shift=1.0), _rand(hd, seed=3, shift=1.0)
    one = torch.ones((), device="cuda", dtype=t)
    packed = _rand(3, 20, 3, 4, hd, seed=4, t=t)
    axis = _rand(2, 20, 5, 3, 4, hd, seed=5, t=t)
    wide = _rand(3, 20, 6, hd + 3, seed=6, t=t)
    for q, k in (
        packed.unbind(2)[:2],
        [x.transpose(1, 2) for x in axis.unbind(3)[:2]],
        (_rand(3, 4, 20, hd, seed=7, t=t).transpose(1, 2), packed[:, :, 1]),
        (wide[..., :hd], wide[..., 3:]),
        (wide[..., 1:hd + 1], wide[:, :, ::2, 2:hd + 2]),
        (wide[:, :, :1, :hd].expand(3, 20, 4, hd), wide[:1, :, :, :hd].expand(3, 20, 6, hd)),
        (_rand(3, 20, 4, 2 * hd, seed=8, t=t)[..., ::2], packed[:, :, 1]),
        (_rand(3, 20, hd, 4, seed=9, t=t).transpose(-1, -2), packed[:, ::1, 2]),
    ):
        for interleaved in (True, False):
            _check_rotary(q, k, f, None, interleaved, dq=one.expand(q.shape), dk=one.expand(k.shape))
            _check_norm(q, k, gq, gk, f, None, interleaved, dq=one.expand(q.shape))


@pytest.mark.parametrize("interleaved", [True, False])
def test_positions(interleaved):
    """Rows of their own, shared ones, 32 and 64 bits, negative, the same twice, strided."""
    f = training.rotary_freqs(32, device="cuda")
    q, k = _rand(4, 2, 30, 4, 40, seed=1), _rand(4, 2, 30, 1, 40, seed=2)
    g = torch.Generator(device="cuda").manual_seed(3)
    each = torch.randint(-(1 << 20), 1 << 20, (4, 2, 30), device="cuda", generator=g)
    each[1] = each[0]
    for p in (each, each.int(), each[0, 0], each[0, 0].int(), each.transpose(0, 1).contiguous().transpose(0, 1),
              torch.zeros_like(each), torch.randint(0, 99, (60,), device="cuda", generator=g)[::2]):
        _check_rotary(q, k, f, p, interleaved)
        _check_norm(q, k, None, None, f, p, interleaved)
    rows = torch.arange(30, device="cuda")
    a, b = training.rotary_forward(q, k, f, rows, interleaved), training.rotary_forward(q, k, f, None, interleaved)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_far_positions():
    """Integers up to 2^53 turn by their exact angle (rational arithmetic), whatever the frequency's type."""
    at = [0, 1, 2**24 - 1, 2**24 + 1, 2**31 - 1, 2**31 + 5, 123456789012345, 2**53 - 1, -(2**53 - 1), -(2**40) - 3]
    for f in (training.rotary_freqs(16), torch.tensor([1.0, 3.7, 1e-3, 1e-9, 100.0, 0.1, 2.0, 1e-15])):
        pos = torch.tensor(at, device="cuda")
        q = torch.zeros(1, len(at), 1, 16, device="cuda")
        q[..., 0::2] = 1.0
        y = training.rotary_forward(q, None, f.cuda(), pos)[0][0, :, 0].double().cpu()
        want = torch.tensor([[w for x in f.tolist() for w in (math.cos(exact_angle(p, x)), math.sin(exact_angle(p, x)))]
                             for p in at], dtype=F64)
        assert_within("far", y, want, torch.full_like(want, TURN))


def test_behind_the_pairs_nothing_changes():
    """Infinities, NaN and negative zeros behind the pairs come through as they are, and reach no pair."""
    for hd, pairs in ((64, 5), (64, 8), (50, 7)):
        f = _rand(pairs, seed=1)
        for interleaved in (True, False):
            q = _rand(1, 9, 2, hd, seed=2)
            q[..., 2 * pairs:] = torch.tensor([math.inf, -math.inf, math.nan, -0.0, 1.0], device="cuda").repeat(20)[:hd - 2 * pairs]
            y, _ = training.rotary_forward(q, None, f, None, interleaved, 3.0)
            assert torch.equal(y[..., 2 * pairs:].nan_to_num(7.0), q[..., 2 * pairs:].nan_to_num(7.0))
            assert torch.equal(torch.signbit(y[..., 2 * pairs:]), torch.signbit(q[..., 2 * pairs:])) or q.isnan().any()
            assert y[..., :2 * pairs].isfinite().all()


@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("hd,pairs", [(64, 32), (50, 20)])
def test_padded_batch(hd, pairs, t):
    """Rows behind the lengths are not used: NaN and infinities there change nothing, and those rows are 0."""
    f, gq, gk = _rand(pairs, seed=1), _rand(hd, seed=2, shift=1.0), _rand(hd, seed=3, shift=1.0)
    q, k = _rand(7, 33, 4, hd, seed=4, t=t), _rand(7, 33, 2, hd, seed=5, t=t)
    dq, dk = _rand(7, 33, 4, hd, seed=6, t=t), _rand(7, 33, 2, hd, seed=7, t=t)
    lens = torch.tensor([33, 0, 1, 32, 17, -5, 99], device="cuda", dtype=torch.int32)
    for eps in (1e-6, 0.0):
        out, back = _check_norm(q, k, gq, gk, f, eps=eps, lens=lens, dq=dq, dk=dk)
        behind = torch.arange(33, device="cuda") >= lens[:, None]
        junk = [x.clone() for x in (q, k, dq, dk)]
        for x, v in zip(junk, (math.nan, math.inf, math.nan, -math.inf)):
            x[behind] = v
        args = (gq, gk, f, None, True, 1.0, eps, lens)
        out2 = training.qk_norm_rotary_forward(junk[0], junk[1], *args)
        back2 = training.qk_norm_rotary_backward(junk[2], junk[3], junk[0], junk[1], *args)
        for a, b in zip((*out, *back), (*out2, *back2)):
            assert torch.equal(a, b)
        assert not any(x[behind].any() for x in (*out2, *back2[:2]))


@pytest.mark.parametrize("interleaved", [True, False])
def test_axial_lengths_and_scales(interleaved):
    """Lengths of (outer, inner) sequences whose token axes are transposed; factors of 0 and below."""
    f, w = _rand(9, seed=1), _rand(48, seed=2, shift=1.0)
    axis = _rand(2, 21, 3, 2, 4, 48, seed=3, t=BF16)
    q, k = (x.transpose(1, 2) for x in axis.unbind(3))
    lens = torch.tensor([21, 0, 5, 20, 1, 13], device="cuda", dtype=torch.int32)
    for scale in (0.0, -1.5, 1e-3):
        _check_norm(q, k, w, w, f, None, interleaved, scale, lens=lens)
        _check_norm(q, None, w, None, f, None, interleaved, scale, lens=lens)
        _check_rotary(q, k, f, None, interleaved, scale)


def test_norm_hard_rows():
    """Rows of zeros, tiny and huge rows; NaN and infinities stay in their row, but for the weights' gradient."""
    f, gq = _rand(32, seed=1), _rand(64, seed=2, shift=1.0)
    q = _rand(1, 9, 2, 64, seed=3)
    q[0, 1], q[0, 2], q[0, 3] = 0.0, q[0, 2] * 1e-9, q[0, 3] * 1e15
    out, back = _check_norm(q, None, gq, None, f)
    assert not out[0][0, 1].any()
    bad = q.clone()
    bad[0, 5, 0, 7], bad[0, 6, 1, 9] = math.nan, math.inf
    dq = _rand(*q.shape, seed=91)
    y, _ = training.qk_norm_rotary_forward(bad, None, gq, None, f)
    dx, _, dg, _ = training.qk_norm_rotary_backward(dq, None, bad, None, gq, None, f)
    for got, clean in ((y, out[0]), (dx, back[0])):
        assert got[0, 5, 0].isnan().all() and got[0, 6, 1].isnan().any()
        got[0, 5, 0], got[0, 6, 1] = clean[0, 5, 0], clean[0, 6, 1]
        assert torch.equal(got, clean)
    assert dg.isnan().any()


def test_weights_of_one_side():
    q, k = _rand(2, 9, 4, 64, seed=1), _rand(2, 9, 2, 64, seed=2)
    f, w = _rand(32, seed=3), _rand(64, seed=4, shift=1.0)
    for gq, gk in ((w, None), (None, w), (None, None)):
        _check_norm(q, k, gq, gk, f)
    got = training.qk_norm_rotary_backward(q, k, q, k, w, w, f, weight_grads=False)
    assert got[2] is None and got[3] is None
    _check_norm(q, k, w, w, None)  # the norm alone


def test_empty():
    f, w = _rand(4, seed=1), torch.ones(8, device="cuda")
    for shape, ks in (((0, 5, 2, 8), (0, 5, 1, 8)), ((2, 0, 2, 8), (2, 0, 2, 8)), ((2, 5, 0, 8), (2, 5, 0, 8))):
        q, k = torch.zeros(shape, device="cuda"), torch.zeros(ks, device="cuda")
        assert [x.shape for x in training.rotary_forward(q, k, f)] == [q.shape, k.shape]
        got = training.qk_norm_rotary_backward(q, k, q, k, w, w, f)
        assert [x.shape for x in got[:2]] == [q.shape, k.shape] and not got[2].any() and not got[3].any()
    q, k = torch.zeros(2, 5, 0, 8, device="cuda"), _rand(2, 5, 3, 8, seed=2)
    _check_rotary(q, k, f)
    _check_norm(q, k, w, w, f)
    _check_rotary(k, q, f)
    _check_norm(k, q, w, w, f)


def test_many_rows():
    """More tokens than teams in flight, and rows beyond 2^31 elements (offsets of 64 bits)."""
    f = training.rotary_freqs(128, device="cuda")
    q = torch.empty(1, (1 << 31) // 256 + 3, 2, 128, device="cuda", dtype=BF16)
    q[:, -5:] = _rand(1, 5, 2, 128, seed=1, t=BF16)
    q[:, :5] = _rand(1, 5, 2, 128, seed=2, t=BF16)
    n = q.shape[1]
    y, _ = training.rotary_forward(q, None, f, None, False)
    for at in (slice(0, 5), slice(n - 5, n)):
        pos = torch.arange(n, device="cuda")[at]
        assert_within("rows", y[:, at], *rotary_reference(q[:, at], f, pos, False, 1.0, False))
    wide = torch.empty(3, 1 << 23, 128, device="cuda", dtype=BF16)  # a stride of 2^30 elements
    wide[:, :7] = _rand(3, 7, 128, seed=3, t=BF16)
    _check_norm(wide[:, :7, None], None, None, None, f)


@pytest.mark.parametrize("interleaved", [True, False])
def test_gradients_by_differences(interleaved):
    """The gradients against central differences of the definition in 64 bits, along random directions."""
    f = _rand(20, seed=1, t=F64)
    q, d = _rand(2, 11, 3, 48, seed=2), _rand(2, 11, 3, 48, seed=3)
    gamma, dgam, dy = _rand(48, seed=4, shift=1.0), _rand(48, seed=5), _rand(2, 11, 3, 48, seed=6)
    got = training.qk_norm_rotary_backward(dy, None, q, None, gamma, None, f, None, interleaved, 1.5)
    ref = qk_norm_reference(q, dy, gamma, f, None, interleaved, 1.5, 1e-6, None)

    def loss(h, dx, dg):
        x, w = q.double() + h * dx, gamma.double() + h * dg
        y = x / ((x * x).mean(-1, keepdim=True) + 1e-6).sqrt() * w
        return rotary_reference(y, f, None, interleaved, 1.5, False)[0].mul(dy.double()).sum()

    zero = torch.zeros((), device="cuda")
    h = 2.0**-17  # cut off after the second order: about h^2; rounding 2^-52 / h of the loss
    for dx, dg, mine, tol in ((d, zero, got[0], ref["dx"][1]), (zero, dgam, got[2], ref["dgamma"][1])):
        slope = (loss(h, dx, dg) - loss(-h, dx, dg)) / (2 * h)
        w = d if mine.dim() == 4 else dgam
        slack = (tol * w.abs()).sum() + 1e-8 * (mine.double() * w).abs().sum()
        assert abs(float((mine.double() * w).sum() - slope)) <= float(slack)


def test_autograd_and_lazy_signs():
    f, gq, gk = _rand(16, seed=1), _rand(32, seed=2, shift=1.0), _rand(32, seed=3, shift=1.0)
    q0, k0 = _rand(2, 9, 4, 32, seed=4), _rand(2, 9, 2, 32, seed=5)
    q, k = q0.clone().requires_grad_(), k0.clone().requires_grad_()
    gq.requires_grad_(), gk.requires_grad_()
    a, b = training.rotary(q, k, f)
    (a.sum() - 2 * b.sum()).backward()
    want = training.rotary_backward(torch.ones_like(q0), torch.full_like(k0, -2.0), f)
    assert torch.equal(q.grad, want[0]) and torch.equal(k.grad, want[1])
    a, b = training.rotary(q, k, f)
    assert torch.equal(torch.autograd.grad(b.sum(), k)[0], training.rotary_backward(torch.ones_like(k0), None, f)[0])
    a, b = training.rotary(q.detach(), k, f)
    assert torch.equal(torch.autograd.grad((a * b.sum()).sum(), k)[0].isfinite().all(), torch.tensor(True, device="cuda"))
    a, b = training.qk_norm_rotary(q, k, gq, gk, f)
    w = _rand(2, 9, 4, 32, seed=6)
    got = torch.autograd.grad((a * w).sum() + b.sum(), (q, k, gq, gk))
    want = training.qk_norm_rotary_backward(w, torch.ones_like(k0), q0, k0, gq.detach(), gk.detach(), f)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    a, b = training.qk_norm_rotary(q, k, gq, gk, f)  # an output that nothing uses, and a weight alone
    got = torch.autograd.grad(a.sum(), (q, gk), allow_unused=True)
    assert got[0] is not None and not got[1].any()
    z = torch.complex(w, w).conj().imag  # negated lazily
    assert z.is_neg()
    a, _ = training.rotary(q, k, f)
    assert torch.equal(torch.autograd.grad(a, q, z)[0], training.rotary_backward(z.resolve_neg(), None, f)[0])
    with pytest.raises(ValueError, match="resolve_neg"):
        training.rotary_forward(z, None, f)
    with pytest.raises(RuntimeError, match="differentiat"):
        a, _ = training.rotary(q, k, f)
        g, = torch.autograd.grad(a.square().sum(), q, create_graph=True)
        g.sum().backward()
    with torch.autograd.forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        training.rotary(torch.autograd.forward_ad.make_dual(q0, q0), k, f)


def test_streams_and_graphs():
    """A side stream, and two graphs that replay in turn on inputs changed in place."""
    f, w = training.rotary_freqs(64, device="cuda"), _rand(64, seed=1, shift=1.0)
    q, k = _rand(2, 100, 4, 64, seed=2, t=BF16), _rand(2, 100, 2, 64, seed=3, t=BF16)
    dq, dk = _rand(2, 100, 4, 64, seed=4, t=BF16), _rand(2, 100, 2, 64, seed=5, t=BF16)
    lens = torch.tensor([100, 60], device="cuda", dtype=torch.int32)
    pos = torch.arange(100, device="cuda")

    def step():
        return (*training.rotary_forward(q, k, f, pos), *training.rotary_backward(dq, dk, f, pos),
                *training.qk_norm_rotary_forward(q, k, w, w, f, pos, lens=lens),
                *training.qk_norm_rotary_backward(dq, dk, q, k, w, w, f, pos, lens=lens))

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step())
        graphs.append(graph)
    for round_ in range(3):
        q.copy_(_rand(2, 100, 4, 64, seed=10 + round_, t=BF16))
        pos.add_(7)
        lens[1] = 10 * round_
        want = step()
        for graph, out in zip(graphs, outs):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))
    x = q.clone().requires_grad_()
    y = training.rotary(x, k, f)[0].sum()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="captured"):
            training.rotary(x, k, f)
        with pytest.raises(RuntimeError, match="captured"):
            training.qk_norm_rotary(x, k, w, w, f)
        torch.zeros(1, device="cuda")
    y.backward()
    assert x.grad is not None


@pytest.mark.parametrize("t", [F32, BF16])
def test_in_front_of_attention(t):
    """Packed projection, norm and rotation, attention, and back: gradients of the projection and the weights against
    64 bits. The largest relative error of a step is a few roundings of each of its five stages."""
    n, length, h, hd = 2, 130, 4, 64
    f = training.rotary_freqs(hd, device="cuda")
    qkv = _rand(n, length, 3, h, hd, seed=1, t=t).requires_grad_()
    gq, gk = (_rand(hd, seed=s, scale=0.2, shift=1.0).requires_grad_() for s in (2, 3))
    dout = _rand(n, length, h, hd, seed=4, t=t)
    lens = torch.tensor([length, 77], device="cuda", dtype=torch.int32)
    q, k, v = qkv.unbind(2)
    q, k = training.qk_norm_rotary(q, k, gq, gk, f, lens=lens)
    out = training.attention(q, k, v, q_lens=lens, k_lens=lens)
    got = (out, *torch.autograd.grad(out, (qkv, gq, gk), dout))

    x = qkv.detach().double().requires_grad_()
    a, b = (g.detach().double().requires_grad_() for g in (gq, gk))
    qd, kd, vd = x.unbind(2)
    qd, kd = ((y / ((y * y).mean(-1, keepdim=True) + 1e-6).sqrt() * w) for y, w in ((qd, a), (kd, b)))
    qd, kd = (rotary_reference(y, f, None, True, 1.0, False)[0] for y in (qd, kd))
    row = torch.arange(length, device="cuda")
    see = (row < lens[:, None])
    z = torch.einsum("nihd,njhd->nhij", qd, kd) * hd**-0.5
    z = z.masked_fill(~see[:, None, None], -math.inf)
    o = torch.einsum("nhij,njhd->nihd", z.softmax(-1), vd) * see[..., None, None]
    want = (o.detach(), *torch.autograd.grad(o, (x, a, b), dout.double()))
    for y, w in zip((x.detach() for x in got), want):
        # five stages, each rounding its operands and result to t; sums of many roundings average out
        rel = float((y.double() - w).norm() / w.norm())
        assert rel <= 10 * half(t) + 2e-6, rel
    assert _lib.error_flag() == 0


def test_one_side_and_the_same_tensor_twice():
    f, w = _rand(16, seed=1), _rand(32, seed=2, shift=1.0).requires_grad_()
    q = _rand(2, 9, 4, 32, seed=3).requires_grad_()
    d = _rand(2, 9, 4, 32, seed=4)
    y, none = training.rotary(q, None, f)
    assert none is None
    assert torch.equal(torch.autograd.grad(y, q, d)[0], training.rotary_backward(d, None, f)[0])
    y, none = training.qk_norm_rotary(q, None, w, None, f)
    assert none is None
    want = training.qk_norm_rotary_backward(d, None, q.detach(), None, w.detach(), None, f)
    got = torch.autograd.grad(y, (q, w), d)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[2])
    a, b = training.rotary(q, q, f)
    assert torch.equal(a, b)
    once = training.rotary_backward(d, None, f)[0]
    assert torch.equal(torch.autograd.grad(a, q, d, retain_graph=True)[0], once)
    assert torch.equal(torch.autograd.grad((a * d).sum() + (b * d).sum(), q)[0], once + once)


def test_two_calls_at_once():
    """Threads with streams of their own."""
    import threading

    f, w = training.rotary_freqs(64, device="cuda"), _rand(64, seed=1, shift=1.0)
    data = [[_rand(3, 500, h, 64, seed=10 * i + h, t=BF16) for h in (4, 2)] for i in range(4)]

    def run(q, k):
        return training.qk_norm_rotary_backward(q, k, q, k, w, w, f)

    want = [run(*d) for d in data]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                got = run(*data[i])
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_packed_parameters():
    """The parameters that a call passes: sizes, strides and addresses of what it was given."""
    q, k = torch.zeros(2, 3, 5, 4, 16, device="cuda")[:, 1:], torch.zeros(2, 2, 5, 2, 18, device="cuda")[..., :16]
    f, pos = torch.ones(8, dtype=F64, device="cuda"), torch.zeros(2, 2, 5, dtype=torch.int64, device="cuda")
    w, lens = torch.ones(16, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    dq, dk = torch.zeros(q.shape, device="cuda"), torch.zeros(k.shape, device="cuda")
    args = (dq, dk, w, None, f, pos, False, 0.5, 1e-3, lens, q, k)
    q_out, k_out, dgq, dgk, at, p, held = _lib.tensor_lists().heads(*args, True, training._norm_workspace())
    assert at == tuple(x.data_ptr() for x in (dq, dk, q, k, q_out, k_out, dgq, dgk, held[-1]))
    assert held[-1].numel() >= 2 * 16 * 4
    assert _lib.tensor_lists().heads(*args, False, training._norm_workspace())[2:4] == (None, None)
    p = _lib.RotaryParams.from_buffer_copy(p)
    got = {n: getattr(p, n) for n, _ in p._fields_ if n not in ("q", "k", "q0", "k0")}
    assert got.pop("eps") == pytest.approx(1e-3)
    assert got == dict(dtype=0, outer=2, inner=2, length=5, heads=4, k_heads=2, hd=16, pairs=8, half=1, scale=0.5,
                       freqs=f.data_ptr(), freqs_f64=1, positions_i64=1, positions=pos.data_ptr(), positions_stride=5,
                       gamma_q=w.data_ptr(), gamma_k=None, w_dtype=0, lens=lens.data_ptr())
    strides = [tuple(getattr(getattr(p, n), m) for m in ("outer", "inner", "row", "head"))
               for n in ("q", "k", "q0", "k0")]
    assert strides == [(640, 320, 64, 16), (320, 160, 32, 16), (960, 320, 64, 16), (360, 180, 36, 18)]
