"""Calls of the training operators at the edge of what they allow, on the GPU against their 64-bit definitions."""

from __future__ import annotations


import pytest
import torch

from training_reference import assert_within, attention_reference, norm_reference
from unblend_b200 import _lib, training

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _rand(*shape, seed, t=F32, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * scale).to(t)


def _attn(n, lq, lk, h, hk, hd, t, seed=0):
    return (_rand(n, lq, h, hd, seed=seed, t=t), _rand(n, lk, hk, hd, seed=seed + 1, t=t),
            _rand(n, lk, hk, hd, seed=seed + 2, t=t), _rand(n, lq, h, hd, seed=seed + 3, t=t))


def test_norm_statistics_inside_a_larger_buffer():
    """``stats`` on either 4-byte boundary gives the gradients that the forward's own tensor gives."""
    x, dy, gamma = _rand(37, 200, seed=1), _rand(37, 200, seed=2), _rand(200, seed=3)
    y, stats = training.layer_norm_forward(x, gamma)
    want = training.layer_norm_backward(dy, x, stats, gamma)
    for at in (0, 1, 2, 3):
        buf = torch.zeros(37 * 2 + 4, device="cuda")
        view = buf[at:at + 74].view(37, 2)
        view.copy_(stats)
        for a, b in zip(training.layer_norm_backward(dy, x, view, gamma), want):
            assert torch.equal(a, b)
    for name, got in (("dx", want[0]), ("dgamma", want[1])):
        assert_within(name, got.reshape(norm_reference(x, gamma, None, 1e-5, dy)[name][0].shape),
                      *norm_reference(x, gamma, None, 1e-5, dy)[name])


@pytest.mark.parametrize("t", [BF16, F16])
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_calls_end_with_everything_used(hd, t):
    """CTAs whose last unit leaves any number of tiles in their rings (none, one, fewer and more than the ring holds):
    many calls behind one another, none of which may find what the one before left."""
    lk = 1200
    kl = torch.tensor([0, 1, 128, 129, 256, 400, 512, 640, 900, lk], device="cuda", dtype=torch.int32)
    q, k, v, dout = _attn(10, 130, lk, 2, 1, hd, t)
    first = None
    for _ in range(20):
        out, lse = training.attention_forward(q, k, v, k_lens=kl)
        got = (out, *training.attention_backward(dout, q, k, v, out, lse, k_lens=kl))
        first = first or [x.clone() for x in got]
        assert all(torch.equal(a, b) for a, b in zip(got, first))
    none = torch.zeros_like(kl)
    out, lse = training.attention_forward(q, k, v, k_lens=none)
    assert not out.any() and not any(x.any() for x in training.attention_backward(dout, q, k, v, out, lse, k_lens=none))
    assert _lib.error_flag() == 0
    ref = attention_reference(q, k, v, dout, k_lens=kl)
    for name, x in zip(("out", "dq", "dk", "dv"), first):
        assert_within(name, x, *ref[name])


# ------------------------------------------------------------------------------- weights of masked keys


@pytest.mark.parametrize("t", [BF16, F16])
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_masked_keys_have_no_weight(hd, t):
    """Values of the type's largest size at keys that a causal query does not see leave its row as it is, bit for bit:
    a weight of 2^-126 in their place would add up to 4 in bf16."""
    q, k, v, _ = _attn(1, 400, 400, 1, 1, hd, t)
    clean, lse = training.attention_forward(q, k, v, causal=True)
    big = v.clone()
    big[:, 350:] = torch.finfo(t).max
    out, lse2 = training.attention_forward(q, k, big, causal=True)
    assert torch.equal(out[:, :350], clean[:, :350]) and torch.equal(lse, lse2)


# ------------------------------------------------------------------------------------------- rows of NaN


@pytest.mark.parametrize("t", [F32, BF16, F16])
@pytest.mark.parametrize("n,lq,lk", [(1, 100, 900), (40, 100, 900), (1, 2, 3000), (3, 40, 50)])
def test_attention_rows_of_nan_say_so(n, lq, lk, t):
    """A query of NaN has an output and a log-sum of NaN, however its keys are divided, and no other row has."""
    q, k, v, dout = _attn(n, lq, lk, 2, 2, 64, t)
    clean, clean_lse = training.attention_forward(q, k, v)
    q[0, 1, 1, 5] = float("nan")
    out, lse = training.attention_forward(q, k, v)
    assert out[0, 1, 1].isnan().all() and lse[0, 1, 1].isnan()
    clean[0, 1, 1], clean_lse[0, 1, 1] = out[0, 1, 1], lse[0, 1, 1]
    assert torch.equal(out.nan_to_num(7.0), clean.nan_to_num(7.0))
    assert torch.equal(lse.nan_to_num(7.0), clean_lse.nan_to_num(7.0))
    dq, _, _ = training.attention_backward(dout, q, k, v, out, lse)
    assert dq[0, 1, 1].isnan().all() and not dq[0, 0].isnan().any() and not dq[0, 1, 0].isnan().any()


# ------------------------------------------------------------------------------------------ blocks of keys


@pytest.mark.parametrize("lq,lk,cut,h,hk,hd", [(60, 64, 60, 2, 2, 64), (40, 64, 60, 4, 2, 64), (30, 36, 32, 2, 2, 64),
                                               (50, 64, 60, 2, 2, 128)])
def test_a_block_of_little_weight_and_large_values(lq, lk, cut, h, hk, hd):
    """The last keys hold about 2^-17.5 of a row's weight, and values a million times larger than the others: D of the
    joined output is mostly theirs, in the gradients of the first block too."""
    q, k, v, dout = _attn(2, lq, lk, h, hk, hd, BF16)
    q, k = q * 0.3, k * 0.3
    q[..., 0], k[..., 0] = hd**0.5, 0.0
    k[:, cut:, :, 0] = -(17.5 * 0.6931 + torch.tensor((lk - cut) / cut).log().item())
    v[:, cut:] *= 1e6
    out, lse = training.attention_forward(q, k, v)
    ref = attention_reference(q, k, v, dout)
    parts = [training.attention_backward(dout, q, k[:, s], v[:, s], out, lse) for s in (slice(0, cut), slice(cut, lk))]
    for i, name in ((1, "dk"), (2, "dv")):
        assert_within(name, torch.cat([x[i] for x in parts], 1), *ref[name])
    want, tol = ref["dq"]
    each = 2.0**-8 * sum(x[0].double().abs() for x in parts)
    assert_within("dq", parts[0][0].double() + parts[1][0].double(), want, tol + each)


@pytest.mark.parametrize("t", [BF16, F16])
@pytest.mark.parametrize("lq,lk,h,hk,hd,causal", [(62, 62, 2, 2, 64, False), (50, 64, 4, 2, 64, True),
                                                  (64, 40, 2, 2, 128, True), (20, 30, 2, 2, 48, False),
                                                  (150, 200, 2, 1, 64, True)])
def test_all_keys_gives_the_same_gradients(lq, lk, h, hk, hd, causal, t):
    """``all_keys`` (D of short sequences from the probabilities), and the differentiable function, which says so."""
    q, k, v, dout = _attn(3, lq, lk, h, hk, hd, t)
    ref = attention_reference(q, k, v, dout, causal=causal)
    out, lse = training.attention_forward(q, k, v, causal=causal)
    got = training.attention_backward(dout, q, k, v, out, lse, causal=causal, all_keys=True)
    for name, x in zip(("dq", "dk", "dv"), got):
        assert_within(name, x, *ref[name])
    leaves = [x.clone().requires_grad_() for x in (q, k, v)]
    training.attention(*leaves, causal=causal).backward(dout)
    assert all(torch.equal(x.grad, y) for x, y in zip(leaves, got))


# --------------------------------------------------------------------------------- sizes of fp16 gradients


def _relative(got, want):
    return float((got.double() - want).norm() / want.norm())


def _fp16_gradients(q, k, v, dout, **kw):
    """Relative error of each gradient next to what rounding its exact value to fp16 costs (subnormals included).

    dS and P are rounded once more on the way, by half a step of 2^-11 each, and so is the output that D is made from;
    errors that do not all point one way add up to less than the sum of both, doubled here.
    """
    out, lse = training.attention_forward(q, k, v, **kw)
    got = training.attention_backward(dout, q, k, v, out, lse, **kw)
    assert _lib.error_flag() == 0
    ref = attention_reference(q, k, v, dout, **kw)
    for name, x in zip(("dq", "dk", "dv"), got):
        want = ref[name][0]
        least = _relative(want.half(), want)
        assert _relative(x, want) <= 2 * (least + 2.0**-11), (name, _relative(x, want), least)


@pytest.mark.parametrize("size", [1.0, 1e-2, 1e-3, 1e-4])
@pytest.mark.parametrize("lq,lk,h,hk,hd,causal", [
    (512, 1344, 1, 1, 64, False), (512, 8192, 1, 1, 64, False), (700, 2000, 2, 1, 128, True),
    (300, 60, 2, 1, 64, False),
    (50, 700, 2, 2, 64, False), (62, 62, 2, 2, 64, False), (64, 50, 4, 2, 48, True), (30, 31, 2, 2, 64, False),
    (60, 60, 2, 2, 128, False), (20, 30, 4, 1, 40, True)])
def test_fp16_gradients_of_small_losses(lq, lk, h, hk, hd, causal, size):
    """Gradients as small as a loss averaged over tokens gives: dS = P (dP - D) must not sink into the subnormals."""
    q, k, v, dout = _attn(2, lq, lk, h, hk, hd, F16, seed=lk)
    _fp16_gradients(q, k, v, (dout.float() * size).half(), causal=causal)


@pytest.mark.parametrize("lq,lk,hd", [(70, 90, 64), (40, 60, 64), (30, 20, 64), (150, 200, 128)])
def test_fp16_gradients_of_scaled_losses(lq, lk, hd):
    """A loss scaled up: dS beyond fp16's largest value, the gradients within it."""
    q, k, v, dout = _attn(2, lq, lk, 1, 1, hd, F16)
    _fp16_gradients(q * 8, k * 8, v * 30, torch.sign(dout) * 500, scale=1 / hd)


def test_fp16_gradients_of_uneven_sequences():
    """Sequences whose gradients differ by 10^6, rows that differ by 10^3, lengths, and NaN behind them."""
    q, k, v, dout = _attn(3, 300, 500, 2, 1, 64, F16)
    dout = dout.float() * torch.tensor([1e-4, 100.0, 1e-2], device="cuda")[:, None, None, None]
    dout[:, ::2] *= 1e-3
    dout = dout.half()
    ql = torch.tensor([300, 200, 77], device="cuda", dtype=torch.int32)
    kl = torch.tensor([500, 333, 450], device="cuda", dtype=torch.int32)
    for b in range(3):
        q[b, int(ql[b]):], dout[b, int(ql[b]):] = float("nan"), float("inf")
        k[b, int(kl[b]):], v[b, int(kl[b]):] = float("nan"), float("inf")
    for b in range(3):
        s = slice(b, b + 1)
        _fp16_gradients(q[s], k[s], v[s], dout[s], q_lens=ql[s], k_lens=kl[s])
    out, lse = training.attention_forward(q, k, v, q_lens=ql, k_lens=kl)
    got = training.attention_backward(dout, q, k, v, out, lse, q_lens=ql, k_lens=kl)
    ref = attention_reference(q, k, v, dout, q_lens=ql, k_lens=kl)
    for b in range(3):
        for name, x in zip(("dq", "dk", "dv"), got):
            want = ref[name][0][b]
            assert _relative(x[b], want) <= 2 * (_relative(want.half(), want) + 2.0**-11), (b, name)
        # The small rows of dq on their own.
        want = ref["dq"][0][b, :int(ql[b]):2]
        assert _relative(got[0][b, :int(ql[b]):2], want) <= 2 * (_relative(want.half(), want) + 2.0**-11), b


@pytest.mark.parametrize("lq,lk,h,hk", [(200, 300, 4, 2), (50, 60, 4, 4), (25, 30, 4, 2)])
def test_infinite_gradients_stay_in_their_head(lq, lk, h, hk):
    """An overflow in one head's dout leaves the scale, and every bit, of the others as they are."""
    q, k, v, dout = _attn(3, lq, lk, h, hk, 64, F16)
    out, lse = training.attention_forward(q, k, v)
    clean = training.attention_backward(dout, q, k, v, out, lse)
    bad = dout.clone()
    bad[1, 7, h - 1, 3] = float("inf")
    got = training.attention_backward(bad, q, k, v, out, lse)
    for x, y in zip(got, clean):
        assert torch.equal(x[[0, 2]], y[[0, 2]]) and torch.equal(x[1, :, 0], y[1, :, 0])
    assert not got[0][1, 7, h - 1].isfinite().any() and not got[1][1, :, hk - 1].isfinite().all()


def test_fp16_passes_captured_and_replayed():
    """Graphs of fp16 passes (long rows, one tile, a few tokens of shared heads) replay on two streams at once, with new
    inputs of another size."""
    shapes = [(2, 200, 300, 4, 2, 64), (20, 50, 60, 4, 4, 64), (20, 20, 30, 4, 2, 48), (1, 500, 700, 4, 1, 128)]

    def step(s):
        out, lse = training.attention_forward(*s[:3])
        return (out, *training.attention_backward(s[3], *s[:3], out, lse))

    sets = [[list(_attn(*c, F16, seed=10 * n + i)) for i, c in enumerate(shapes)] for n in range(2)]
    for s in sets[1]:
        s[3] *= 1e-3
    want = [[[x.clone() for x in step(s)] for s in group] for group in sets]
    held = [[x.clone() for x in s] for s in sets[0]]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append([step(s) for s in held])
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    for n in (0, 1, 0):
        for mine, new in zip(held, sets[n]):
            for x, y in zip(mine, new):
                x.copy_(y)
        torch.cuda.synchronize()
        for _ in range(5):
            for graph, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    graph.replay()
        torch.cuda.synchronize()
        for got in outs:
            for a, b in zip(got, want[n]):
                assert all(torch.equal(x, y) for x, y in zip(a, b))
    assert _lib.error_flag() == 0


def test_calls_run_on_the_current_stream_without_torchs_private_handle(monkeypatch):
    """The stream's handle comes from a function that torch does not document; without it the public one serves."""
    x = _rand(500, 64, seed=5)
    want = training.layer_norm_forward(x)[0].clone()
    side = torch.cuda.Stream()
    for gone in (False, True):
        if gone:
            monkeypatch.delattr(torch._C, "_cuda_getCurrentRawStream", raising=False)
            monkeypatch.setattr(_lib, "_raw_stream", None)
            monkeypatch.setattr(_lib, "current_device", torch.cuda.current_device)
        for stream in (torch.cuda.current_stream(), side):
            with torch.cuda.stream(stream):
                assert _lib.current_stream() == stream.cuda_stream
                y = x * 1
                got = training.layer_norm_forward(y)[0]
            stream.synchronize()
            assert torch.equal(got, want)


def test_gradients_that_arrive_as_lazily_negated_views():
    """The gradient of the imaginary part of a conjugated number is a view with its sign beside it: it counts."""
    rng = torch.tensor([5, 6], device="cuda")
    x, w, q = _rand(6, 40, 64, seed=1), _rand(64, seed=2), _rand(2, 30, 4, 64, seed=3)
    weight = torch.complex(_rand(6, 40, 64, seed=4), _rand(6, 40, 64, seed=5))
    qw = torch.complex(_rand(2, 30, 4, 64, seed=6), _rand(2, 30, 4, 64, seed=7))
    calls = ((lambda a: training.layer_norm(a, w), x, weight), (lambda a: training.attention(a, a, a), q, qw),
             (lambda a: training.dropout_add(a, 0.2, rng, a, w), x, weight),
             (lambda a: training.dropout_add(a, 0.2, rng), x, weight))
    for call, inp, wt in calls:
        grads = []
        for lazy in (True, False):
            leaf = inp.clone().requires_grad_()
            y = call(leaf)
            if lazy:  # |(0 + i y)* - wt|^2 / 2 without the square of y: Re(wt * conj(i y)) = Im(wt) y
                (torch.complex(torch.zeros_like(y), y).conj() * wt).real.sum().backward()
            else:
                (y * wt.imag).sum().backward()
            grads.append(leaf.grad)
        assert torch.equal(grads[0], grads[1])
