"""Transformer operators with gradients, for fine-tuning the separation models.

Three operators of the models' pre-norm block ``x + LayerScale * dropout(attention(layer_norm(x)))``
(unblend/transformer.py:290-301, 328-359; unblend/roformer.py:478-511), each as

* a differentiable function (``layer_norm``, ``attention``, ``dropout_add``), and
* its two passes as plain calls (``*_forward``, ``*_backward``) for callers that keep the saved tensors themselves.

All take CUDA tensors in fp32, bf16 or fp16 and run hand-written kernels on the current stream of the tensors' device;
wrong arguments raise ``ValueError`` before anything is launched, and there is no CPU path. Statistics, softmax and
sums are fp32 whatever the type. No result depends on scheduling: two calls on the same inputs agree bit for bit.
Memory is allocated by torch for each call, so calls on several streams and captured graphs share nothing.

The attention kernels on the tensor cores wait for one another's steps with a limit of two seconds. A wait that runs out
leaves the outputs unfinished and sets a flag on the device, which no call reads (that would wait for the GPU): read
``_lib.error_flag()`` where a step is checked anyway; it is 0 unless something is wrong.

CUDA graphs: capture the plain calls. The differentiable functions refuse to record or run a backward pass while a
stream is being captured: autograd's gradient accumulation of leaves that an earlier eager pass still holds runs on
that pass's stream, which breaks the capture. Second derivatives and forward-mode derivatives are refused too.
"""

from __future__ import annotations

import ctypes
import math
from functools import lru_cache

import torch
from torch.autograd import forward_ad

from . import _lib

_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}
MAX_HEAD_DIM = 128
_F32_MAX = torch.finfo(torch.float32).max
_REGISTER_COLS = 8192  # widest rows whose layer norm sums the weights' gradients beside the input's
_MOST = 1 << 31  # rows, and columns, of layer norm and dropout-add


def _launch(t: torch.Tensor, name: str, *args, kernels: int = 1) -> None:
    """Calls an entry point, which launches ``kernels`` kernels, on the current stream of ``t``'s device."""
    if _lib.current_device() == t.get_device():
        _lib.call(name, *args, kernels=kernels)
    else:
        with torch.cuda.device(t.get_device()):
            _lib.call(name, *args, kernels=kernels)


def _empty(like: torch.Tensor, dtype: torch.dtype | None = None) -> torch.Tensor:
    if dtype is None and like.is_contiguous():
        return torch.empty_like(like)
    return torch.empty_like(like, dtype=dtype, memory_format=torch.contiguous_format)


def _check_tensor(name: str, t, like: torch.Tensor | None = None) -> None:
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a tensor, got {type(t).__name__}")
    if t.dtype not in _DTYPES:
        raise ValueError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    if t.is_neg():  # the memory holds the other sign
        raise ValueError(f"{name} is a lazily negated view: give {name}.resolve_neg()")
    if like is not None and t.device != like.device:
        raise ValueError(f"{name} is on {t.device}, expected {like.device}")


def _check_rows(x: torch.Tensor) -> None:
    if x.shape[-1] >= _MOST or x.numel() >= _MOST * x.shape[-1]:
        raise ValueError(f"x must have fewer than 2^31 rows and columns, got shape {tuple(x.shape)}")


def _check_cuda(name: str, t: torch.Tensor) -> None:
    """Last of the checks, so that the others answer on machines without a GPU too."""
    if not t.is_cuda:
        raise ValueError(f"{name} is on {t.device}: the training operators run on CUDA devices only")


def _check_weight(name: str, w, x: torch.Tensor) -> None:
    _check_tensor(name, w, x)
    if w.dtype not in (torch.float32, x.dtype):
        raise ValueError(f"{name} must be float32 or {x.dtype} like its input, got {w.dtype}")
    if w.shape != x.shape[-1:]:
        raise ValueError(f"{name} must have shape ({x.shape[-1]},), got {tuple(w.shape)}")


def _rows(t: torch.Tensor) -> tuple[torch.Tensor, int, int, int, int]:
    """``t`` as rows of its last axis: (tensor, outer, inner, outer stride, inner stride).

    Any layout whose leading axes collapse to two is taken as it is; others are copied.
    """
    if t.is_contiguous():  # the usual case at a fifth of the host time: small calls are bound by it
        cols = t.shape[-1]
        return t, 1, t.numel() // cols, 0, cols
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        t = t.contiguous()
    for _ in range(2):
        dims: list[tuple[int, int]] = []  # (size, stride) of the leading axes, merged where they run on
        for n, s in zip(t.shape[:-1], t.stride()[:-1]):
            if n == 1:
                continue
            if dims and dims[-1][1] == n * s:
                dims[-1] = (dims[-1][0] * n, s)
            else:
                dims.append((n, s))
        if len(dims) <= 2:
            break
        t = t.contiguous()
    while len(dims) < 2:
        dims.insert(0, (1, 0))
    return t, dims[0][0], dims[1][0], dims[0][1], dims[1][1]


def _same_split(a: tuple, b: tuple) -> tuple[tuple, tuple]:
    """Two row layouts of the same shape brought to one (outer, inner) split."""
    if a[1:3] == b[1:3]:
        return a, b

    def cut(r, outer, inner):  # a one-level layout takes any split
        return (r[0], outer, inner, inner * r[4], r[4]) if r[1] == 1 else None

    got = cut(a, *b[1:3])
    if got is not None:
        return got, b
    got = cut(b, *a[1:3])
    if got is not None:
        return a, got
    return _same_split(a, _rows(b[0].contiguous()))


@lru_cache(maxsize=4096)
def _workspace_bytes(name: str, rows: int, cols: int) -> int:
    n = ctypes.c_longlong(0)
    _lib.check(name, getattr(_lib.load(), name)(rows, cols, ctypes.byref(n)))
    return n.value


@lru_cache(maxsize=4096)
def _attention_workspace_bytes(backward: int, *sizes) -> int:
    """Refuses sizes that the kernels do not take, on the way."""
    p = _lib.AttnTrainParams(*sizes)
    n = ctypes.c_longlong(0)
    rc = _lib.ERR_INVALID
    if max(sizes[:-1]) < _MOST:  # the fields are 32 bits
        rc = _lib.load().unblend_attention_workspace(ctypes.byref(p), backward, ctypes.byref(n))
    if rc == _lib.ERR_INVALID:
        raise ValueError("sizes beyond what attention takes: outer {1}, inner {2}, {3} heads over {4}, {5} queries, "
                         "{6} keys, head_dim {7}".format(*sizes))
    _lib.check("unblend_attention_workspace", rc)
    return n.value


def _scratch(t: torch.Tensor, nbytes: int) -> torch.Tensor | None:
    return t.new_empty(nbytes, dtype=torch.uint8) if nbytes else None


def _refuse_capture(what: str) -> None:
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{what} cannot take part in autograd while a CUDA graph is captured; "
                           f"capture {what}_forward and {what}_backward instead")


# ------------------------------------------------------------------------------------------ layer norm


def _check_norm(x, gamma, beta, eps: float) -> None:
    _check_tensor("x", x)
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"x must have a last axis to normalise over, got shape {tuple(x.shape)}")
    _check_rows(x)
    if not (isinstance(eps, (int, float)) and eps >= 0):
        raise ValueError(f"eps must be >= 0, got {eps!r}")
    for name, w in (("gamma", gamma), ("beta", beta)):
        if w is not None:
            _check_weight(name, w, x)
    if gamma is not None and beta is not None and gamma.dtype != beta.dtype:
        raise ValueError(f"gamma and beta must share a type, got {gamma.dtype} and {beta.dtype}")


def layer_norm_forward(x: torch.Tensor, gamma: torch.Tensor | None = None, beta: torch.Tensor | None = None,
                       eps: float = 1e-5) -> tuple[torch.Tensor, torch.Tensor]:
    """Layer norm over the last axis: ``(y, stats)``.

    ``y = (x - mean) * rstd * gamma + beta`` in x's type; ``stats`` (fp32, ``[rows, 2]``) holds each row's mean and
    reciprocal standard deviation for ``layer_norm_backward``. ``gamma`` and ``beta`` are fp32 or x's type, or None.
    """
    _check_norm(x, gamma, beta, eps)
    _check_cuda("x", x)
    y = _empty(x)
    n = x.numel() // x.shape[-1]
    stats = x.new_empty((n, 2), dtype=torch.float32)
    if n == 0:
        return y, stats
    w = gamma if gamma is not None else beta
    gamma = None if gamma is None else gamma.contiguous()
    beta = None if beta is None else beta.contiguous()
    xr, outer, inner, so, si = _rows(x)
    dt = _DTYPES[x.dtype]
    _launch(x, "unblend_layer_norm_forward", xr.data_ptr(), so, si, y.data_ptr(), stats.data_ptr(),
            _lib.ptr(gamma), _lib.ptr(beta), eps, outer, inner, x.shape[-1], dt,
            _lib.DTYPE_F32 if w is None else _DTYPES[w.dtype])
    return y, stats


def layer_norm_backward(dy: torch.Tensor, x: torch.Tensor, stats: torch.Tensor, gamma: torch.Tensor | None = None,
                        weight_grads: bool = True) -> tuple[torch.Tensor, torch.Tensor | None, torch.Tensor | None]:
    """``(dx, dgamma, dbeta)`` from the output's gradient, the input and the forward pass's ``stats``.

    The weights' gradients have gamma's type (fp32 without gamma) and are None with ``weight_grads=False``.
    """
    _check_norm(x, gamma, None, 0.0)
    _check_tensor("dy", dy, x)
    if dy.shape != x.shape or dy.dtype != x.dtype:
        raise ValueError(f"dy must be {x.dtype} of shape {tuple(x.shape)}, got {dy.dtype} {tuple(dy.shape)}")
    n, cols = x.numel() // x.shape[-1], x.shape[-1]
    if not isinstance(stats, torch.Tensor) or stats.shape != (n, 2) or stats.dtype != torch.float32 or \
            stats.device != x.device:
        raise ValueError("stats must be the second result of layer_norm_forward for this x")
    _check_cuda("x", x)
    dx = _empty(x)
    wt = torch.float32 if gamma is None else gamma.dtype
    dgamma = dbeta = None
    if weight_grads:
        dgamma, dbeta = x.new_empty(cols, dtype=wt), x.new_empty(cols, dtype=wt)
    if n == 0:
        return (dx, dgamma.zero_(), dbeta.zero_()) if weight_grads else (dx, None, None)
    if gamma is not None:
        gamma = gamma.contiguous()
    stats = stats.contiguous()
    if stats.data_ptr() % 8:  # a row's two values are one access; a slice of a larger buffer may lie between
        stats = stats.clone()
    (xr, outer, inner, x_so, x_si), (dyr, _, _, d_so, d_si) = _same_split(_rows(x), _rows(dy))
    work = _scratch(x, _workspace_bytes("unblend_layer_norm_grad_workspace", n, cols)) if weight_grads else None
    _launch(x, "unblend_layer_norm_backward", dyr.data_ptr(), d_so, d_si, xr.data_ptr(), x_so, x_si,
            stats.data_ptr(), _lib.ptr(gamma), dx.data_ptr(), _lib.ptr(dgamma), _lib.ptr(dbeta),
            _lib.ptr(work), outer, inner, cols, _DTYPES[x.dtype], _DTYPES[wt],
            kernels=1 + (work is not None) + (weight_grads and cols > _REGISTER_COLS))
    return dx, dgamma, dbeta


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gamma, beta, eps):
        y, stats = layer_norm_forward(x, gamma, beta, eps)
        ctx.save_for_backward(x, gamma, stats)
        ctx.beta_dtype = None if beta is None else beta.dtype
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        _refuse_capture("layer_norm")
        x, gamma, stats = ctx.saved_tensors
        need_w = ctx.needs_input_grad[1] or ctx.needs_input_grad[2]
        dx, dgamma, dbeta = layer_norm_backward(dy.resolve_neg(), x, stats, gamma, need_w)
        if not ctx.needs_input_grad[1]:
            dgamma = None
        dbeta = dbeta.to(ctx.beta_dtype) if ctx.needs_input_grad[2] else None
        return dx, dgamma, dbeta, None


def _wants_grad(what: str, *tensors) -> bool:
    """Whether a call has to be recorded; tangents of forward mode, which no operator here carries on, are refused."""
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{what} has no forward-mode derivative")
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def layer_norm(x: torch.Tensor, gamma: torch.Tensor | None = None, beta: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """Differentiable layer norm over the last axis (``layer_norm_forward`` / ``layer_norm_backward``)."""
    _check_norm(x, gamma, beta, eps)
    if _wants_grad("layer_norm", x, gamma, beta):
        _check_cuda("x", x)
        _refuse_capture("layer_norm")
        return _LayerNorm.apply(x, gamma, beta, eps)
    return layer_norm_forward(x, gamma, beta, eps)[0]


# ------------------------------------------------------------------------------------------- attention


def _check_heads(name: str, t, like: torch.Tensor | None = None) -> None:
    _check_tensor(name, t, like)
    if t.dim() not in (4, 5):
        raise ValueError(f"{name} must be [batch, length, heads, head_dim] or [outer, inner, length, heads, head_dim], "
                         f"got shape {tuple(t.shape)}")
    if like is not None and t.dtype != like.dtype:
        raise ValueError(f"{name} must be {like.dtype} like q, got {t.dtype}")


def _check_lens(name: str, lens, seqs: int, q: torch.Tensor) -> None:
    if lens is None:
        return
    if not isinstance(lens, torch.Tensor) or lens.dtype != torch.int32 or lens.device != q.device:
        raise ValueError(f"{name} must be an int32 tensor on {q.device}")
    if lens.numel() != seqs:
        raise ValueError(f"{name} must hold one length for each of {seqs} sequences, got {lens.numel()}")


def _check_attention(q, k, v, scale, causal, q_lens, k_lens) -> float:
    _check_heads("q", q)
    _check_heads("k", k, q)
    _check_heads("v", v, q)
    if k.shape != v.shape:
        raise ValueError(f"k and v must have one shape, got {tuple(k.shape)} and {tuple(v.shape)}")
    if k.dim() != q.dim() or k.shape[:-3] != q.shape[:-3] or k.shape[-1] != q.shape[-1]:
        raise ValueError(f"q {tuple(q.shape)} and k {tuple(k.shape)} must agree in their batch axes and head_dim")
    if q.shape[-2] == 0 or k.shape[-2] == 0 or q.shape[-2] % k.shape[-2]:
        raise ValueError(f"{q.shape[-2]} query heads must be a multiple of {k.shape[-2]} key/value heads")
    if not 1 <= q.shape[-1] <= MAX_HEAD_DIM:
        raise ValueError(f"head_dim must be 1 to {MAX_HEAD_DIM}, got {q.shape[-1]}")
    seqs = _seqs(q)
    _check_lens("q_lens", q_lens, seqs, q)
    _check_lens("k_lens", k_lens, seqs, q)
    scale = q.shape[-1] ** -0.5 if scale is None else float(scale)
    if not abs(scale) <= _F32_MAX:
        raise ValueError(f"scale must be finite in float32, got {scale}")
    return scale


def _unit(t: torch.Tensor) -> torch.Tensor:
    return t if t.shape[-1] == 1 or t.stride(-1) == 1 else t.contiguous()


def _strides(t: torch.Tensor) -> _lib.HeadStrides:
    s = t.stride()
    return _lib.HeadStrides(s[0], s[1] if len(s) == 5 else 0, s[-3], s[-2])


def _sizes(q, k, scale: float, causal: bool) -> tuple:
    """The leading fields of ``AttnTrainParams``."""
    s, lk, kv_heads = q.shape, k.shape[-3], k.shape[-2]
    return (_DTYPES[q.dtype], s[0], s[1] if len(s) == 5 else 1, s[-2], kv_heads, s[-3], lk, s[-1], bool(causal),
            scale)


def _seqs(q) -> int:
    return q.shape[0] if q.dim() == 4 else q.shape[0] * q.shape[1]


def attention_forward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float | None = None,
                      causal: bool = False, q_lens: torch.Tensor | None = None,
                      k_lens: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Multi-head attention ``softmax(scale q k^T) v``: ``(out, lse)``.

    q is ``[batch, lq, heads, head_dim]`` or, for axial sequences, ``[outer, inner, lq, heads, head_dim]``; k and v
    likewise with lk and their own number of heads, which divides q's (head h of q reads head ``h // (heads //
    kv_heads)``). Any strides with a unit last one are taken as they are: slices of one packed projection, transposed
    token axes. ``scale`` defaults to ``head_dim ** -0.5``; head_dim is at most 128. 16-bit calls run on the tensor cores
    when head_dim is a multiple of 8, ``scale`` positive, and every tensor starts, and strides along each axis of more
    than one, by a positive multiple of 16 bytes; others (keys expanded over heads: give the shared head itself) run on
    the CUDA cores, many times slower.

    ``q_lens`` / ``k_lens`` (int32, one per sequence) are the sequences' lengths in a padded batch; rows behind them
    are not used, whatever they hold. With ``causal``, query i sees keys ``j <= i + k_len - q_len``. Queries that see
    no key and rows behind q_len come out as 0 with ``lse = -inf``. ``out`` is contiguous in q's type and shape;
    ``lse`` (fp32, ``[sequences, heads, lq]``) is what ``attention_backward`` recomputes the probabilities from.
    """
    scale = _check_attention(q, k, v, scale, causal, q_lens, k_lens)
    empty = q.numel() == 0 or k.shape[-3] == 0
    sizes = _sizes(q, k, scale, causal)
    n = 0 if empty else _attention_workspace_bytes(0, *sizes)
    _check_cuda("q", q)
    out = _empty(q)
    lse = q.new_empty((_seqs(q), q.shape[-2], q.shape[-3]), dtype=torch.float32)
    if empty:
        return out.zero_(), lse.fill_(-math.inf)
    q, k, v = _unit(q), _unit(k), _unit(v)
    q_lens = None if q_lens is None else q_lens.contiguous()
    k_lens = None if k_lens is None else k_lens.contiguous()
    p = _lib.AttnTrainParams(*sizes, _lib.ptr(q_lens), _lib.ptr(k_lens), _strides(q), _strides(k), _strides(v),
                             _strides(out))
    work = _scratch(q, n)
    _launch(q, "unblend_attention_forward", q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.data_ptr(),
            _lib.ptr(work), n, ctypes.byref(p))
    return out, lse


def attention_backward(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                       lse: torch.Tensor, scale: float | None = None, causal: bool = False,
                       q_lens: torch.Tensor | None = None, k_lens: torch.Tensor | None = None,
                       all_keys: bool = False) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``(dq, dk, dv)`` from the gradient of ``out``, the inputs and the results of ``attention_forward``.

    The probabilities are computed again from q, k and ``lse``; dk and dv are summed over the query heads that share a
    head. The gradients are contiguous; rows behind the lengths are 0. Keys that are processed in blocks may give each
    block ``out`` and ``lse`` of all of them: dk and dv are then the block's rows, and the blocks' dq add up.
    ``all_keys=True`` says that this call is not such a block: 16-bit sequences of up to 64 queries and keys then take
    ``rowsum(dout * out)`` from the fp32 probabilities, without the rounding of ``out``, and do not read ``out``.
    """
    scale = _check_attention(q, k, v, scale, causal, q_lens, k_lens)
    for name, t in (("dout", dout), ("out", out)):
        _check_heads(name, t, q)
        if t.shape != q.shape:
            raise ValueError(f"{name} must have q's shape {tuple(q.shape)}, got {tuple(t.shape)}")
    seqs = _seqs(q)
    if not isinstance(lse, torch.Tensor) or lse.shape != (seqs, q.shape[-2], q.shape[-3]) or \
            lse.dtype != torch.float32 or lse.device != q.device:
        raise ValueError("lse must be the second result of attention_forward for this q")
    empty = q.numel() == 0 or k.numel() == 0
    sizes = _sizes(q, k, scale, causal)
    n = 0 if empty else _attention_workspace_bytes(1, *sizes)
    _check_cuda("q", q)
    dq, dk, dv = _empty(q), _empty(k), _empty(v)
    if empty:
        return dq.zero_(), dk.zero_(), dv.zero_()
    q, k, v, out, dout = _unit(q), _unit(k), _unit(v), _unit(out), _unit(dout)
    q_lens = None if q_lens is None else q_lens.contiguous()
    k_lens = None if k_lens is None else k_lens.contiguous()
    p = _lib.AttnTrainParams(*sizes, _lib.ptr(q_lens), _lib.ptr(k_lens),
                             *(_strides(t) for t in (q, k, v, out, dout, dq, dk, dv)), bool(all_keys))
    lse = lse.contiguous()
    work = _scratch(q, n)
    _launch(q, "unblend_attention_backward", dout.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(),
            out.data_ptr(), lse.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _lib.ptr(work), n,
            ctypes.byref(p))
    return dq, dk, dv


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, scale, causal, q_lens, k_lens):
        out, lse = attention_forward(q, k, v, scale, causal, q_lens, k_lens)
        ctx.save_for_backward(q, k, v, out, lse, q_lens, k_lens)
        ctx.scale, ctx.causal = scale, causal
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        _refuse_capture("attention")
        q, k, v, out, lse, q_lens, k_lens = ctx.saved_tensors
        dq, dk, dv = attention_backward(dout.resolve_neg(), q, k, v, out, lse, ctx.scale, ctx.causal, q_lens, k_lens,
                                        all_keys=True)
        need = ctx.needs_input_grad
        return dq if need[0] else None, dk if need[1] else None, dv if need[2] else None, None, None, None, None


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float | None = None, causal: bool = False,
              q_lens: torch.Tensor | None = None, k_lens: torch.Tensor | None = None) -> torch.Tensor:
    """Differentiable multi-head attention (arguments as ``attention_forward``)."""
    scale = _check_attention(q, k, v, scale, causal, q_lens, k_lens)
    if _wants_grad("attention", q, k, v):
        _check_cuda("q", q)
        _refuse_capture("attention")
        return _Attention.apply(q, k, v, scale, causal, q_lens, k_lens)
    return attention_forward(q, k, v, scale, causal, q_lens, k_lens)[0]


# ----------------------------------------------------------------------------------------- dropout-add


def _check_dropout(x, p: float, rng, residual, scale) -> None:
    _check_tensor("x", x)
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"x must have a last axis, got shape {tuple(x.shape)}")
    _check_rows(x)
    if not (isinstance(p, (int, float)) and 0 <= p <= 1):
        raise ValueError(f"p must be a probability, got {p!r}")
    if not isinstance(rng, torch.Tensor) or rng.dtype != torch.int64 or rng.numel() != 2 or rng.device != x.device:
        raise ValueError(f"rng must be an int64 tensor (seed, offset) on {x.device}")
    if scale is not None:
        _check_weight("scale", scale, x)
    if residual is not None:
        _check_tensor("residual", residual, x)
        if residual.shape != x.shape or residual.dtype not in (torch.float32, x.dtype):
            raise ValueError(f"residual must be float32 or {x.dtype} of shape {tuple(x.shape)}, got {residual.dtype} "
                             f"{tuple(residual.shape)}")


def dropout_add_forward(x: torch.Tensor, p: float, rng: torch.Tensor, residual: torch.Tensor | None = None,
                        scale: torch.Tensor | None = None) -> torch.Tensor:
    """``residual + scale * dropout(x, p)``, kept values divided by ``1 - p``.

    ``rng`` (int64, ``(seed, offset)``, on x's device) picks the mask: element e of x in row-major order is kept when
    word ``e % 4`` of Philox-4x32-10 with key ``seed`` and counter ``(e // 4, offset)`` is at least ``round(p *
    2**32)``. The mask is not stored: give ``dropout_add_backward`` the same ``rng``, and each dropout of a step its
    own offset. A dropped element adds exactly nothing, whatever it holds. ``scale`` (LayerScale, ``[cols]``) is fp32
    or x's type; the result has the residual's type (fp32 or x's), or x's without one.
    """
    _check_dropout(x, p, rng, residual, scale)
    _check_cuda("x", x)
    t = x.dtype if residual is None else residual.dtype
    y = _empty(x) if t == x.dtype else _empty(x, t)
    if x.numel() == 0:
        return y
    rng = rng.contiguous()
    scale = None if scale is None else scale.contiguous()
    xr = _rows(x)
    rr = (None, 1, 1, 0, 0)
    if residual is not None:
        xr, rr = _same_split(xr, _rows(residual))
    _launch(x, "unblend_dropout_add_forward", xr[0].data_ptr(), xr[3], xr[4], _lib.ptr(rr[0]), rr[3], rr[4],
            _lib.ptr(scale), y.data_ptr(), float(p), rng.data_ptr(), xr[1], xr[2], x.shape[-1], _DTYPES[x.dtype],
            _DTYPES[t], _lib.DTYPE_F32 if scale is None else _DTYPES[scale.dtype])
    return y


def dropout_add_backward(dy: torch.Tensor, x: torch.Tensor, p: float, rng: torch.Tensor,
                         scale: torch.Tensor | None = None, scale_grad: bool = True
                         ) -> tuple[torch.Tensor, torch.Tensor | None]:
    """``(dx, dscale)`` of ``dropout_add_forward`` with the same ``p``, ``rng`` and ``scale``.

    dy (fp32 or x's type) is the residual's gradient as it is. dscale has scale's type, and is None without a scale or
    with ``scale_grad=False``.
    """
    _check_dropout(x, p, rng, None, scale)
    _check_tensor("dy", dy, x)
    if dy.shape != x.shape or dy.dtype not in (torch.float32, x.dtype):
        raise ValueError(f"dy must be float32 or {x.dtype} of shape {tuple(x.shape)}, got {dy.dtype} "
                         f"{tuple(dy.shape)}")
    _check_cuda("x", x)
    return _dropout_backward(dy, x, x.dtype, p, rng, scale, scale is not None and scale_grad)


def _dropout_backward(dy, x, dtype, p: float, rng, scale, scale_grad: bool):
    """The backward pass of checked arguments; x, of type ``dtype``, is read only with ``scale_grad``."""
    dx = _empty(dy) if dy.dtype == dtype else _empty(dy, dtype)
    dscale = _empty(scale) if scale_grad else None
    if dy.numel() == 0:
        return dx, None if dscale is None else dscale.zero_()
    rng = rng.contiguous()
    scale = None if scale is None else scale.contiguous()
    dr = _rows(dy)
    xr = (None, dr[1], dr[2], 0, 0)
    work = None
    if scale_grad:
        dr, xr = _same_split(dr, _rows(x))
        work = _scratch(dy, _workspace_bytes("unblend_dropout_add_grad_workspace", dr[1] * dr[2], dy.shape[-1]))
    _launch(dy, "unblend_dropout_add_backward", dr[0].data_ptr(), dr[3], dr[4], _lib.ptr(xr[0]), xr[3], xr[4],
            _lib.ptr(scale), dx.data_ptr(), _lib.ptr(dscale), _lib.ptr(work), float(p), rng.data_ptr(), dr[1], dr[2],
            dy.shape[-1], _DTYPES[dtype], _DTYPES[dy.dtype],
            _lib.DTYPE_F32 if scale is None else _DTYPES[scale.dtype], kernels=1 + scale_grad)
    return dx, dscale


class _DropoutAdd(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, rng, residual, scale):
        # The backward pass draws the mask again: it keeps a copy, so that the caller may advance rng in place.
        rng = rng.clone()
        ctx.save_for_backward(x if scale is not None and ctx.needs_input_grad[4] else None, rng, scale)
        ctx.p, ctx.residual, ctx.dtype = p, residual is not None, x.dtype
        return dropout_add_forward(x, p, rng, residual, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        _refuse_capture("dropout_add")
        x, rng, scale = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx = dscale = None
        if need[0] or need[4]:
            dx, dscale = _dropout_backward(dy.resolve_neg(), x, ctx.dtype, ctx.p, rng, scale, need[4])
        return dx if need[0] else None, None, None, dy if ctx.residual and need[3] else None, dscale


def dropout_add(x: torch.Tensor, p: float, rng: torch.Tensor, residual: torch.Tensor | None = None,
                scale: torch.Tensor | None = None) -> torch.Tensor:
    """Differentiable ``residual + scale * dropout(x, p)`` (arguments as ``dropout_add_forward``)."""
    _check_dropout(x, p, rng, residual, scale)
    if _wants_grad("dropout_add", x, residual, scale):
        _check_cuda("x", x)
        _refuse_capture("dropout_add")
        return _DropoutAdd.apply(x, p, rng, residual, scale)
    return dropout_add_forward(x, p, rng, residual, scale)
