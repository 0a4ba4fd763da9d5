"""What AdamW refuses beyond wrong shapes: memory that a step would write and use at the same time. No GPU needed."""

from __future__ import annotations

import ctypes
from array import array

import pytest
import torch

from unblend_b200 import _lib, training

step = training.adamw_step


def _refused(params, grads, state, number=1, **kw):
    with pytest.raises(ValueError, match="share memory"):
        step(params, grads, state, number, **kw)


def _accepted(params, grads, state, number=1, **kw):
    with pytest.raises(ValueError, match="CUDA devices only"):  # the last of the checks
        step(params, grads, state, number, **kw)


def test_moments_share_no_memory():
    p = [torch.zeros(300)]
    buf = torch.zeros(1024)
    for m, v in ((buf[:512], buf[256:768]), (buf[256:768], buf[:512]), (buf[:512], buf[:512]), (buf[:512], buf[508:1020])):
        _refused(p, p, training.AdamWState(m, v))
        with pytest.raises(ValueError, match="share memory"):
            training.adamw_moments(training.AdamWState(m, v))
    _accepted(p, [torch.zeros(300)], training.AdamWState(buf[:512], buf[512:]))
    raw = torch.zeros(2048, dtype=torch.uint8)
    m, v = raw[:512], raw[512:1024]
    for at in (0, 496, 504, 512, 1008):
        _refused(p, p, training.AdamWState(m, v, raw[at:at + 16].view(torch.float32).view(2, 2)))
    _accepted(p, [torch.zeros(300)], training.AdamWState(m, v, raw[1024:1040].view(torch.float32).view(2, 2)))


@pytest.mark.parametrize("bits", [32, 8])
def test_tensors_share_no_memory_with_the_state(bits):
    p, g = [torch.zeros(300), torch.zeros(7)], [torch.zeros(300), torch.zeros(7)]
    s = training.adamw_state(p, bits)
    for flat in s:
        if flat is None:
            continue
        raw = flat.view(-1).view(torch.float32)
        for x in (raw[:2], raw[-2:], raw[1:4]):
            own = torch.zeros(x.numel())
            _refused([x, p[0]], [own, None], training.AdamWState(*s))
            _refused([own, p[0]], [x, None], training.AdamWState(*s))
            _refused([p[0], own.half()], [None, x], training.AdamWState(*s))
            _refused([p[0], x], [g[0].half(), own.half()], training.AdamWState(*s))  # two pairs of types in one call
            _accepted([p[0], x], [g[0], None], training.AdamWState(*s))  # not written
    if bits == 32:
        _refused(p, training.adamw_views(p, s.exp_avg), s)
    _accepted(p, g, s)


def test_numbers_on_the_device_share_no_memory_with_what_is_written():
    p, g = [torch.zeros(300), torch.zeros(8)], [torch.zeros(300), torch.zeros(8)]
    s = training.adamw_state(p, 8)
    for x in (p[0], p[1], s.scales.view(-1), s.exp_avg.view(torch.float32), s.exp_avg_sq.view(torch.float32)):
        _refused(p, g, s, lr=x[2:3])
        _refused(p, g, s, grad_scale=x[-1:])
        _refused(p, g, s, x[2:4].view(torch.int64))
    _accepted(p, g, s, lr=g[0][:1], grad_scale=g[1][3:4])
    _refused(p, [torch.zeros(300).half(), g[1]], s, lr=p[0][5:6])


def test_entry_point_refuses_shared_moments():
    """Nothing is launched: every call is refused."""
    lib = _lib.load()
    x = ctypes.create_string_buffer(1 << 16)
    p = (ctypes.addressof(x) + 15) & ~15
    far = p + (1 << 40)  # addresses are compared, not read

    def call(rows, m, v, s=None, bits=32, **kw):
        t = array("q", [w for r in rows for w in r])
        a = _lib.AdamWParams(1e-3, 0.9, 0.999, 1e-8, 0.01, 1)
        for n, w in kw.items():
            setattr(a, n, w)
        return lib.unblend_adamw_step(t.buffer_info()[0], len(rows), m, v, s, bits, 0, 0, ctypes.byref(a), None)

    one, two = [(p, p + 4096, 300, 0)], [(p, p + 4096, 300, 0), (p + 2048, p + 8192, 10, 2)]
    for rows, m, v in ((one, far, far), (one, far, far + 2032), (one, far + 2032, far), (one, p, far), (one, far, p + 1184),
                       (one, p + 4096, far), (one, far, p + 4096 - 2032),
                       (two, far, far + 2048), (two[::-1], far, far + 3056),  # the third block of one is the other's
                       ([two[0], (p + 2048, p + 8192, 10, 1)], far, far + 65536),  # two tensors in one block
                       ([two[0], (p + 2048, p + 8192, 10, 0)], far, far + 65536),
                       ([(p + 2048, p + 8192, 10, 1), two[0]], far, far + 65536)):
        assert call(rows, m, v) == _lib.ERR_OVERLAP
    for m, v, s in ((far, far + 512, far), (far, far + 512, far + 504), (far, far + 512, far + 1016), (far, far + 496, p),
                    (far, far + 512, p + 8), (far, far + 512, p + 4096), (far, far + 512, p + 4096 - 8)):
        assert call(one, m, v, s, 8) == _lib.ERR_OVERLAP
    for n in ("step_device", "lr_device", "grad_scale"):
        for at in (p, p + 1192, far, far + 2040, far + 65536 + 8):
            assert call(one, far, far + 65536, **{n: at}) == _lib.ERR_OVERLAP
        assert call(one, far, far + 512, far + 4096, 8, **{n: far + 4096 + 8}) == _lib.ERR_OVERLAP
    assert call([(p, p + 4096, 300, 1 << 31)], far, far + 65536) == _lib.ERR_INVALID


def test_clipping_to_what_fp32_does_not_hold():
    """Below the smallest fp32 number a largest norm would be 0."""
    g = [torch.ones(5)]
    for bad in (1e-46, 5e-324, -1e-50):
        with pytest.raises(ValueError, match="max_norm must be"):
            training.grad_norm(g, bad)
    for good in (1e-45, 3e38, 1):
        with pytest.raises(ValueError, match="CUDA devices only"):
            training.grad_norm(g, good)
