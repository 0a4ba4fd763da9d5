"""AdamW over many tensors and the norm of gradients on the GPU against their 64-bit definitions."""

from __future__ import annotations

import math

import pytest
import torch

from adamw_reference import M_TABLE, U_TABLE, adamw_reference, codes, values
from training_reference import U, assert_within
from unblend_b200 import training

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
SIZES = [(1,), (3,), (16, 16), (255,), (257,), (5, 200), (64, 64), (0,), (331, 211), (2, 128), ()]
ARGS = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.05)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _model(seed, t=F32, tg=None, sizes=SIZES):
    g = _gen(seed)
    params = [(torch.randn(s, device="cuda", generator=g) * 0.3).to(t) for s in sizes]
    grads = [(torch.randn(s, device="cuda", generator=g) * 10.0 ** (-3 + i % 4)).to(tg or t) for i, s in enumerate(sizes)]
    return params, grads


def _pad(flat_parts, sizes):
    out = []
    for x in flat_parts:
        n = x.numel()
        out.append(torch.nn.functional.pad(x.reshape(-1).float(), (0, -n % 256)))
    return torch.cat(out)


def _state(params, bits, seed):
    """A state as after some steps: moments of many sizes, zeros behind the parameters."""
    g = _gen(seed)
    state = training.adamw_state(params, bits)
    m = _pad([torch.randn(p.shape, device="cuda", generator=g) * 10.0 ** (-4 + i % 3) for i, p in enumerate(params)],
             None)
    u = _pad([torch.randn(p.shape, device="cuda", generator=g).exp() * 10.0 ** (-4 + i % 3)
              for i, p in enumerate(params)], None)
    if bits == 32:
        return training.AdamWState(m, u * u)
    (cm, tm), (cu, tu) = codes(m, M_TABLE), codes(u, U_TABLE)
    assert state.exp_avg.shape == cm.shape and state.scales.shape == (len(tm), 2)
    return training.AdamWState(cm, cu, torch.stack((tm, tu), 1))


def _values(state):
    if state.scales is None:
        return state.exp_avg.clone(), state.exp_avg_sq.clone()
    u = values(state.exp_avg_sq, state.scales[:, 1], U_TABLE)
    return values(state.exp_avg, state.scales[:, 0], M_TABLE), u * u


def _check_step(params, grads, state, step=7, gs=0.75, **kw):
    """One step against the definition, tensor by tensor; returns the parameters as they were."""
    kw = {**ARGS, **kw}
    old = [p.clone() for p in params]
    m0, v0 = _values(state)
    if state.scales is not None:
        got = training.adamw_moments(state)
        assert torch.equal(got[0], m0) and torch.equal(got[1], v0)
    scale = torch.tensor(gs, device="cuda")
    training.adamw_step(params, grads, state, step, grad_scale=scale, **kw)
    m1, v1 = training.adamw_moments(state)
    views = [training.adamw_views(params, x) for x in (m0, v0, m1, v1)]
    args = (step, kw["lr"], kw["betas"], kw["eps"], kw["weight_decay"], gs)
    want_m, want_u = [], []
    for i, (p, g) in enumerate(zip(params, grads)):
        if g is None:
            assert torch.equal(p, old[i])
            continue
        ref, m32, u32 = adamw_reference(old[i], g, views[0][i], views[1][i], *args)
        assert_within(f"p[{i}]", p, *ref["p"])
        if state.scales is None:
            assert_within(f"m[{i}]", views[2][i], *ref["m"])
            assert_within(f"v[{i}]", views[3][i], *ref["v"])
        want_m.append(m32), want_u.append(u32)
    if state.scales is not None and all(g is not None for g in grads):
        (cm, tm), (cu, tu) = codes(_pad(want_m, None), M_TABLE), codes(_pad(want_u, None), U_TABLE)
        assert torch.equal(state.scales, torch.stack((tm, tu), 1))
        same = (cm == state.exp_avg) | ((cm & 127 == 0) & (state.exp_avg & 127 == 0))
        assert bool(same.all()) and torch.equal(cu, state.exp_avg_sq)
    return old


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("tg", [F32, BF16, F16])
def test_types(tg, t, bits):
    params, grads = _model(1, t, tg)
    state = _state(params, bits, 2)
    for step in (1, 2, 1000):
        _check_step(params, grads, state, step)
    _check_step(params, grads, training.adamw_state(params, bits), 1)  # from zeros
    _check_step(params, grads, state, 10**6, lr=0.0)
    _check_step(params, grads, state, 3, betas=(0.0, 0.0), weight_decay=0.0, eps=1.0)


@pytest.mark.parametrize("bits", [32, 8])
def test_unaligned_views_and_gaps(bits):
    """Parameters and gradients anywhere in larger buffers; what lies between them stays."""
    sizes = [1, 300, 256, 1000, 7, 513]
    for t in (F32, BF16):
        buf, gbuf = (torch.randn(4000, device="cuda", generator=_gen(s)).to(t) for s in (3, 4))
        for gap in (1, 2, 3, 4, 8):
            at, params, grads = 1, [], []
            used = torch.zeros(4000, dtype=torch.bool, device="cuda")
            for n in sizes:
                params.append(buf[at:at + n]), grads.append(gbuf[at + 1:at + 1 + n])
                used[at:at + n] = True
                at += n + gap
            before = buf.clone()
            _check_step(params, grads, _state(params, bits, 5))
            assert torch.equal(buf[~used], before[~used]) and not torch.equal(buf, before)


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors(bits):
    """More tensors than one launch takes, in one call, beside tensors of other types and missing gradients."""
    sizes = [(1 + (i * 37) % 400,) for i in range(2000)]
    params, grads = _model(6, sizes=sizes)
    for i in range(0, 2000, 9):
        params[i], grads[i] = params[i].to(BF16), grads[i].to(BF16)
    for i in range(0, 2000, 7):
        grads[i] = None
    state = _state(params, bits, 7)
    before = [x.clone() for x in training.adamw_views(params, state.exp_avg)]
    _check_step(params, grads, state)
    for i in range(0, 2000, 7):
        assert torch.equal(training.adamw_views(params, state.exp_avg)[i], before[i])
    for n in (1, 64, 65, 896, 897):
        _check_step(params[:n], [g if g is not None else torch.zeros_like(p) for p, g in zip(params[:n], grads[:n])],
                    _state(params[:n], bits, 8))
    training.adamw_step(params[:1], [None], _state(params[:1], bits, 8), 1)


@pytest.mark.parametrize("bits", [32, 8])
def test_large_tensor(bits):
    """Work for several rounds of the grid, and (8 bits) elements behind 2^31."""
    n = 30_000_001 if bits == 32 else (1 << 31) + 1001
    p, g = torch.zeros(n, device="cuda", dtype=BF16), torch.zeros(n, device="cuda", dtype=BF16)
    for x, s in ((p, 1), (g, 2)):
        x[-3000:] = torch.randn(3000, device="cuda", generator=_gen(s)).to(BF16)
    state = training.adamw_state([p], bits)
    tail = p[-3000:].clone()
    training.adamw_step([p], [g], state, 1, **ARGS)
    z = torch.zeros(3000, device="cuda")
    ref, _, _ = adamw_reference(tail, g[-3000:], z, z, 1, *ARGS.values(), 1.0)
    assert_within("p", p[-3000:], *ref["p"])
    assert not p[:-3000].any()


@pytest.mark.parametrize("bits", [32, 8])
def test_a_scale_that_is_not_finite_changes_nothing(bits):
    params, grads = _model(9)
    state = _state(params, bits, 10)
    before = [x.clone() for x in (*params, *(y for y in state if y is not None))]
    grads[4][0] = math.inf
    for bad in (math.nan, math.inf, -math.inf):
        training.adamw_step(params, grads, state, 3, grad_scale=torch.tensor(bad, device="cuda"))
    _, scale = training.grad_norm(grads, 1.0)
    training.adamw_step(params, grads, state, 3, grad_scale=scale)
    assert all(torch.equal(a, b) for a, b in zip(before, (*params, *(y for y in state if y is not None))))


def test_values_that_are_not_finite():
    """Without a clipping factor, an infinite gradient spoils its element (32 bits) or its block (8 bits)."""
    for bits in (32, 8):
        for bad in (math.inf, math.nan):
            params, grads = _model(11, sizes=[(256,), (700,)])
            grads[1][300] = bad
            state = _state(params, bits, 12)
            old = [p.clone() for p in params]
            training.adamw_step(params, grads, state, 2)
            assert params[0].isfinite().all() and params[1][300].isnan()
            assert params[1][:300].isfinite().all() and params[1][301:].isfinite().all()
            m, v = (training.adamw_views(params, x)[1] for x in training.adamw_moments(state))
            keep = torch.ones(700, dtype=torch.bool, device="cuda")
            keep[300 if bits == 32 else slice(256, 512)] = False
            assert m[keep].isfinite().all() and v[keep].isfinite().all()
            assert not m[~keep].isfinite().any() and not v[~keep].isfinite().any()
            assert not torch.equal(old[0], params[0])


def test_codes_at_their_borders():
    """Every code, ties between codes, zeros, signs, the smallest codes and values below them, blocks of zeros and of tiny
    values: moments that a step with beta = 0 takes from the gradient as they are."""
    top = 0.75
    for table in (M_TABLE, U_TABLE):
        mid = (table[1:] + table[:-1]) / 2
        near = torch.cat((table, mid, mid * (1 + 2.0**-20), mid * (1 - 2.0**-20), table[1:3] * 0.3, table[1:2] * 1e-9))
        g = torch.cat((near, -near)).float().cuda() * top
        g = torch.cat((g, torch.zeros(-len(g) % 255, device="cuda"))).view(-1, 255)
        g = torch.cat((torch.full((len(g), 1), top, device="cuda"), g), 1)  # the block's largest
        g = torch.cat((g, torch.zeros(1, 256, device="cuda"), torch.full((1, 256), 1e-30, device="cuda"),
                       torch.full((1, 256), 1e-41, device="cuda"), torch.full((1, 256), 3e38, device="cuda") ** 0.5))
        p = [torch.zeros(g.numel(), device="cuda")]
        state = training.adamw_state(p, 8)
        _check_step(p, [g.view(-1)], state, 2, 1.0, betas=(0.0, 0.0), eps=1.0)


def test_steps_and_rates_on_the_device():
    for bits in (32, 8):
        for t in (1, 5, 100000):
            params, grads = _model(13, BF16)
            other = [p.clone() for p in params]
            a, b = _state(params, bits, 14), _state(params, bits, 14)
            training.adamw_step(params, grads, a, t, 0.125, weight_decay=0.25)
            training.adamw_step(other, grads, b, torch.tensor([t], device="cuda"), torch.tensor(0.125, device="cuda"),
                                weight_decay=0.25)
            for x, y in zip((*params, *a[:2]), (*other, *b[:2])):
                assert_within("device", x, y, (2.0**-7 if x.dtype == BF16 else 8 * U) * y.double().abs()
                              if x.dtype != torch.uint8 else torch.zeros(x.shape, device="cuda"))
            training.adamw_step(params, grads, a, t, torch.tensor(0.125, device="cuda"))
            training.adamw_step(other, grads, b, torch.tensor(t, device="cuda"), 0.125)
            for x, y in zip(params, other):
                assert_within("device", x, y, 2.0**-6 * y.double().abs() + 2.0**-20)


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps(bits):
    """Two graphs of a clipped step, replayed in turn with new gradients, steps and rates, beside eager calls; a side
    stream gives the same."""
    params, grads = _model(15)
    eager = [p.clone() for p in params]
    state, other = _state(params, bits, 16), _state(params, bits, 16)
    step, lr = torch.ones((), dtype=torch.int64, device="cuda"), torch.tensor(1e-2, device="cuda")

    def run(p, s):
        _, scale = training.grad_norm(grads, 1.0)
        training.adamw_step(p, grads, s, step, lr, grad_scale=scale)

    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run(params, state)
        graphs.append(graph)
    side = torch.cuda.Stream()
    for n in range(6):
        for i, g in enumerate(grads):
            g.copy_(torch.randn(g.shape, device="cuda", generator=_gen(100 * n + i)))
        step.fill_(n + 1)
        lr.mul_(0.9)
        graphs[n % 2].replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(eager, other)
        torch.cuda.current_stream().wait_stream(side)
        for a, b in zip((*params, *(x for x in state if x is not None)), (*eager, *(x for x in other if x is not None))):
            assert torch.equal(a, b)


def test_shared_memory_is_refused():
    p = torch.zeros(1000, device="cuda")
    g = torch.zeros(1000, device="cuda")
    for params, grads in (([p, p], [g, g]), ([p[:600], p[599:]], [g[:600], g[599:]]), ([p[:500]], [p[400:900]]),
                          ([p[:100], p[50:60]], [g[:100], g[:10]]),
                          ([p[:100], p[50:60].view(BF16)], [g[:100], g[:20].to(BF16)])):
        with pytest.raises(ValueError, match="share memory"):
            training.adamw_step(params, grads, training.adamw_state(params), 1)
    training.adamw_step([p[:500], p[500:]], [g[:500], g[:500]], training.adamw_state([p[:500], p[500:]]), 1)


def test_autograd_sees_the_change():
    p = torch.ones(5, device="cuda", requires_grad=True)
    y = (p * p).sum()
    training.adamw_step([p], [torch.ones(5, device="cuda")], training.adamw_state([p]), 1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


# --------------------------------------------------------------------------------------- norm of gradients


def _check_norm(grads, max_norm=1.0):
    norm, scale = training.grad_norm(grads, max_norm)
    want = math.sqrt(sum(float(g.double().square().sum()) for g in grads if g is not None))
    assert norm.dtype == scale.dtype == F32 and norm.shape == scale.shape == ()
    # 64-bit sums; one rounding each to fp32
    assert abs(float(norm) - want) <= 2 * U * want + 2.0**-149
    f = min(1.0, max_norm / want) if want else 1.0
    assert abs(float(scale) - f) <= 2 * U * f
    again = training.grad_norm(grads, max_norm)
    assert torch.equal(norm, again[0]) and torch.equal(scale, again[1])
    assert training.grad_norm(grads)[1] is None and torch.equal(training.grad_norm(grads)[0], norm)


@pytest.mark.parametrize("t", [F32, BF16, F16])
def test_norm_sizes(t):
    _, grads = _model(20, t)
    _check_norm(grads)
    _check_norm([None, *grads, None], 1e6)
    for n in (1, 31, 1023, 1024, 1025, 8192, 3_000_001):
        g = torch.randn(n + 3, device="cuda", generator=_gen(n)).to(t)
        _check_norm([g[:n]])
        _check_norm([g[3:], g[1:n], g[2:]])  # off 16-byte boundaries; shared memory is only read


def test_norm_of_many_types():
    sizes = [(1 + (i * 53) % 3000,) for i in range(2100)]
    _, grads = _model(21, sizes=sizes)
    grads = [g.to((F32, BF16, F16)[i % 3]) for i, g in enumerate(grads)]
    _check_norm(grads)
    _check_norm(grads[::3][:64] + grads[1::3][:65])


def test_norm_extremes():
    """No overflow or underflow on the way; zeros; values that are not finite."""
    _check_norm([torch.full((1000,), 1e37, device="cuda")], 2.0)
    _check_norm([torch.full((1000,), 1e-37, device="cuda")], 1e-38)
    _check_norm([torch.zeros(5, device="cuda"), torch.zeros(0, device="cuda")])
    for bad in (math.inf, -math.inf, math.nan):
        g = torch.ones(5000, device="cuda")
        g[4321] = bad
        norm, scale = training.grad_norm([g], 1.0)
        assert not norm.isfinite() and scale.isnan()
    norm, scale = training.grad_norm([torch.zeros(0, device="cuda")], 1.0)
    assert float(norm) == 0 and float(scale) == 1


def test_norm_past_32_bits():
    g = torch.zeros((1 << 32) + 77, device="cuda", dtype=F16)
    g[-5:], g[1 << 31] = 2.0, 3.0
    norm, _ = training.grad_norm([g])
    assert abs(float(norm) - math.sqrt(29.0)) <= 2 * U * 6


# ------------------------------------------------------------------------------------------ a whole step


@pytest.mark.parametrize("t", [F32, BF16])
def test_a_training_step(t):
    """Norm, packed projection, norm and rotation of queries and keys, attention, dropout-add and back, then the gradients'
    norm and the update, which is checked against the definition on the gradients that autograd left."""
    n, length, dim, heads = 2, 65, 128, 2
    g = _gen(30)
    f = training.rotary_freqs(64, device="cuda")
    rng = torch.tensor([1, 2], device="cuda")
    params = [(torch.randn(s, device="cuda", generator=g) * 0.1 + b).to(w).requires_grad_()
              for s, b, w in (((dim,), 1.0, F32), ((dim, 3 * dim), 0.0, t), ((64,), 1.0, F32), ((64,), 1.0, F32),
                              ((dim, dim), 0.0, t), ((dim,), 0.5, F32))]
    norm, w_qkv, gq, gk, w_out, ls = params
    x = torch.randn(n, length, dim, device="cuda", generator=g).to(t)
    lens = torch.tensor([length, 40], device="cuda", dtype=torch.int32)
    state = {8: training.adamw_state(params, 8), 32: training.adamw_state(params)}
    for bits in (8, 32):
        for step in (1, 2):
            h = training.layer_norm(x, norm)
            q, k, v = (h @ w_qkv).unflatten(-1, (3, heads, 64)).unbind(-3)
            q, k = training.qk_norm_rotary(q, k, gq, gk, f, lens=lens)
            q, k = training.rotary(q, k, f)
            a = training.attention(q, k, v, q_lens=lens, k_lens=lens).flatten(-2) @ w_out
            y = training.dropout_add(a, 0.1, rng, x, ls)
            grads = torch.autograd.grad(y.float().square().mean(), params)
            total, scale = training.grad_norm(grads, 0.5)
            assert total.isfinite() and float(total) > 0
            _check_step([p.detach() for p in params], list(grads), state[bits], step, float(scale))
            rng[1] += 1
