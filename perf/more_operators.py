"""More operators of ``unblend_b200.training`` as measured calls: rotary positions, the norm of queries and keys with the
rotation in the same pass, AdamW over all parameters of a model, and the norm of all gradients.

``run`` takes one pass through an operator: in elementary torch operations where ``own`` is false, through the
framework's public functions where it is true. ``exact`` gives the same outputs from the definition in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
EPS = 1e-6
BLOCK = 256  # elements of a moment that share a scale; every parameter starts a block of its own
BETAS, ADAM_EPS, DECAY, LR = (0.9, 0.999), 1e-8, 0.01, 3e-4


# ---------------------------------------------------------------------------------------------- cases


def _heads(name, op, outer, inner, length, heads, kv_heads, hd, rot, dtype, pairs="interleaved", layout="split",
           positions="rows", factor=1.0, weights="fp32", ragged=False, backward=True):
    """``layout``: "split" q and k of their own; "packed" column blocks of one projection; "axis" packed, with the
    sequences running along the first of two token axes. ``positions``: "rows" 0, 1, ...; "given" per sequence, each from
    a start of its own. ``rot``: rotated dims (0: the norm alone); ``factor``: how many times longer the context is than
    the frequencies were made for; "ragged": per-sequence lengths in a padded batch."""
    return {"name": name, "op": op, "outer": outer, "inner": inner, "length": length, "heads": heads,
            "kv_heads": kv_heads, "hd": hd, "rot": rot, "dtype": dtype, "pairs": pairs, "layout": layout,
            "positions": positions, "factor": factor, "weights": weights, "ragged": ragged, "backward": backward}


def _model(name, op, layers, dim, bands, dtype, grads, bits=32, step=1000):
    """The parameters of an axial separator: ``layers`` transformer blocks of width ``dim`` and the projections of
    ``bands`` bands. ``bits`` of the moments; ``step``: number of the update."""
    return {"name": name, "op": op, "layers": layers, "dim": dim, "bands": bands, "dtype": dtype, "grads": grads,
            "bits": bits, "step": step}


def listed():
    return [
        # One STFT frame of a 62-band separator in fp32: the smallest call, where launches count.
        _heads("rotary one frame", "rotary", 1, 1, 62, 8, 8, 64, 64, "fp32"),
        # Time axis of an axial model in training: 62 sequences of 801 tokens out of one packed projection, rows far apart.
        _heads("rotary time axis", "rotary", 1, 62, 801, 8, 8, 64, 64, "bf16", layout="axis"),
        # Long odd context beyond the trained one, part of wide heads in the half layout, shared key heads, starts of
        # their own (chunks of long recordings).
        _heads("rotary long partial half", "rotary", 3, 1, 16381, 16, 4, 128, 64, "fp16", "half", positions="given",
               factor=8.0),
        # Streams that add one token each, far into their contexts: forward alone.
        _heads("rotary one token", "rotary", 96, 1, 1, 16, 4, 128, 128, "bf16", "half", positions="given",
               backward=False),
        # Band axis of an axial model: 801 sequences of 62 tokens out of one packed projection.
        _heads("qk norm band axis", "qk_norm", 1, 801, 62, 8, 8, 64, 64, "bf16", layout="packed"),
        # Padded batch of clips with their own lengths (some empty), fp32, 48-wide heads of which 36 dims turn.
        _heads("qk norm padded fp32", "qk_norm", 6, 1, 1343, 8, 8, 48, 36, "fp32", ragged=True),
        # Many tokens of a wide model with shared key heads: bandwidth alone.
        _heads("qk norm many wide tokens", "qk_norm", 2, 1, 40009, 32, 8, 128, 128, "bf16", "half", weights="bf16"),
        # One small layer in fp32: launches count.
        _model("adamw one layer", "adamw", 1, 64, 3, "fp32", "fp32", step=3),
        # All of a 12-layer, 62-band separator in fp32.
        _model("adamw whole model", "adamw", 12, 512, 62, "fp32", "fp32"),
        # A wider one in bf16 with 8-bit moments; the pass hands out the moments' values too.
        _model("adamw bf16 8 bits", "adamw", 18, 640, 60, "bf16", "bf16", bits=8),
        # The norm before the update of the 62-band separator.
        _model("grad norm whole model", "grad_norm", 12, 512, 62, "fp32", "fp32"),
        # A small 16-bit model of odd sizes.
        _model("grad norm small odd", "grad_norm", 2, 93, 7, "fp16", "fp16"),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["rotary", "rotary", "qk_norm", "qk_norm", "adamw", "adamw", "grad_norm"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op in ("adamw", "grad_norm"):
        dim = log(24, 512)
        layers = log(1, 12)
        grads = rng.choice([dtype, dtype, "fp32"]) if op == "adamw" else dtype
        c = _model("", op, layers, dim, log(2, 62), dtype, grads, rng.choice([32, 8]) if op == "adamw" else 32,
                   log(1, 100000))
    else:
        hd = rng.choice([32, 40, 48, 64, 64, 80, 96, 128, 128, 160, 256])
        rot = rng.choice([hd, hd, hd // 2, 2 * (hd // 5)])
        heads = rng.choice([4, 8, 12, 16, 32])
        layout = rng.choice(["split", "split", "packed", "axis"])
        kv = heads if layout != "split" else rng.choice([heads, heads // 2, heads // 4])
        length = log(1, 32768)
        cap = 1 << (26 if dtype == "fp32" else 27)  # elements of q
        length = min(length, cap // (heads * hd))
        batch = max(1, min(log(1, 1024), cap // (heads * hd * length)))
        c = _heads("", op, 1 if layout == "axis" else batch, batch if layout == "axis" else 1, length, heads, kv, hd,
                   rot, dtype, rng.choice(["interleaved", "half"]), layout, rng.choice(["rows", "rows", "given"]),
                   rng.choice([1.0, 1.0, 4.0, 32.0]), rng.choice(["fp32", dtype]),
                   op == "qk_norm" and layout != "axis" and rng.random() < 0.3, rng.random() < 0.8)
    del c["name"]
    return c


# --------------------------------------------------------------------------------------------- inputs


def _freqs(case):
    """Frequencies in radians per position (64 bits) and the factor on the rotated values: for longer contexts the slow
    pairs, which did not turn once within the trained 8192 positions, are slowed down by the factor, those of 32 turns and
    more are kept, and the ones between are mixed."""
    n = case["rot"] // 2
    f = 10000.0 ** (-torch.arange(n, dtype=torch.float64) / max(n, 1))
    if case["factor"] == 1.0:
        return f.cuda(), 1.0
    keep = ((8192 * f / (2 * math.pi) - 1) / 31).clamp(0, 1)
    return (f * keep + f / case["factor"] * (1 - keep)).cuda(), 0.1 * math.log(case["factor"]) + 1


def _prepare_heads(case, g):
    t = DTYPES[case["dtype"]]
    o, i, n, h, hk, hd = (case[m] for m in ("outer", "inner", "length", "heads", "kv_heads", "hd"))

    def rand(*shape):
        return torch.randn(*shape, device="cuda", generator=g).to(t)

    if case["layout"] == "split":
        q, k = rand(o * i, n, h, hd), rand(o * i, n, hk, hd)
    elif case["layout"] == "packed":
        q, k, _ = rand(o * i, n, 3, h, hd).unbind(2)
    else:  # tokens are [outer, sequence position, inner]: the sequences of (outer, inner) run along the middle
        q, k, _ = (x.transpose(1, 2) for x in rand(o, n, i, 3, h, hd).unbind(3))
    s = {"q": q, "k": k, "positions": None, "lens": None, "gamma_q": None, "gamma_k": None}
    s["freqs"], s["scale"] = _freqs(case)
    if case["backward"]:  # as the attention behind them returns them
        s["dq"], s["dk"] = rand(*q.shape), rand(*k.shape)
    if case["positions"] == "given":
        start = torch.randint(0, 1 << 20, (*q.shape[:-3], 1), device="cuda", generator=g)
        s["positions"] = start + torch.arange(n, device="cuda")
    if case["op"] == "qk_norm":
        tw = DTYPES[case["weights"]]
        s["gamma_q"], s["gamma_k"] = ((1 + 0.2 * torch.randn(hd, device="cuda", generator=g)).to(tw) for _ in range(2))
        if case["ragged"]:
            s["lens"] = torch.randint(0, n + 1, (o * i,), device="cuda", generator=g, dtype=torch.int32)
    return s


def _shapes(case):
    dim, bands = case["dim"], case["bands"]
    heads = max(1, dim // 64)
    block = [(dim,), (3 * dim, dim), (heads, dim), (heads,), (dim, dim), (dim,), (4 * dim, dim), (4 * dim,),
             (dim, 4 * dim), (dim,)]
    ends = []
    for b in range(bands):
        width = 8 * (1 + b * b // 64)  # the bands grow towards high frequencies
        ends += [(width,), (dim, width), (dim,), (2 * dim, dim), (2 * dim,), (2 * width, 2 * dim), (2 * width,)]
    return block * (2 * case["layers"]) + [(dim,)] + ends


def _prepare_model(case, g):
    """Parameters and gradients as views of one buffer each, every one from a block of its own; zeros between them."""
    t, tg = DTYPES[case["dtype"]], DTYPES[case["grads"]]
    shapes = _shapes(case)
    sizes = [math.prod(x) for x in shapes]
    blocks = [-(-n // BLOCK) for n in sizes]
    count = torch.tensor(blocks, device="cuda")
    total = sum(blocks)
    first = (count.cumsum(0) - count) * BLOCK
    at = torch.arange(total * BLOCK, device="cuda") - first.repeat_interleave(count).repeat_interleave(BLOCK)
    used = at < torch.tensor(sizes, device="cuda").repeat_interleave(count).repeat_interleave(BLOCK)

    def views(flat):
        return [x[:n].view(d) for x, n, d in zip(flat.split([b * BLOCK for b in blocks]), sizes, shapes)]

    def rand():
        return torch.randn(total * BLOCK, device="cuda", generator=g) * used

    # Gradients of one tensor have one size, those of different tensors have not.
    size = (10.0 ** (-4 + 2 * torch.rand(len(sizes), device="cuda", generator=g))).repeat_interleave(count)
    size = size.repeat_interleave(BLOCK)
    flat_g = (rand() * size).to(tg)
    s = {"flat_g": flat_g, "grads": views(flat_g)}
    if case["op"] == "grad_norm":
        return s
    flat_p = (0.05 * rand()).to(t)
    m, u = rand() * size * 0.3, (rand() * 0.5).exp() * used * size
    s |= {"flat_p": flat_p, "params": views(flat_p), "step": case["step"],
          "grad_scale": torch.rand((), device="cuda", generator=g) * 0.5 + 0.5}
    if case["bits"] == 32:
        return s | {"m": m, "v": u * u, "scales": None}
    top_m, top_u = (x.view(-1, BLOCK).abs().amax(1) for x in (m, u))
    cm, cu = _codes(m, top_m, 7, 3), _codes(u, top_u, 8, 4)
    return s | {"m": cm, "v": cu, "scales": torch.stack((top_m, top_u), 1)}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    make = _prepare_model if case["op"] in ("adamw", "grad_norm") else _prepare_heads
    return {"case": dict(case), **make(case, g)}


# ---------------------------------------------------------------------------------------- plain forms


def _cos_sin(s):
    """[..., length, 1, n]: angles of far positions in 64 bits."""
    p = torch.arange(s["case"]["length"], device="cuda") if s["positions"] is None else s["positions"]
    angle = (p.double()[..., None] * s["freqs"])[..., None, :]
    return (angle.cos() * s["scale"]).float(), (angle.sin() * s["scale"]).float()


def _turn(x, cos, sin, half):
    """x (32 bits) turned pair by pair; dims behind the pairs stay."""
    n = cos.shape[-1]
    if half:
        a, b, rest = x[..., :n], x[..., n:2 * n], x[..., 2 * n:]
        return torch.cat((a * cos - b * sin, a * sin + b * cos, rest), -1)
    a, b, rest = x[..., :2 * n:2], x[..., 1:2 * n:2], x[..., 2 * n:]
    return torch.cat((torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2), rest), -1)


def _plain_rotary(s):
    cos, sin = _cos_sin(s)
    half, t = s["case"]["pairs"] == "half", s["q"].dtype
    res = {m: _turn(s[m].float(), cos, sin, half).to(t) for m in ("q", "k")}
    if s["case"]["backward"]:  # the transposed rotation
        res |= {m: _turn(s[m].float(), cos, -sin, half).to(t) for m in ("dq", "dk")}
    return res


def _plain_qk_norm(s):
    cos, sin = _cos_sin(s)
    case = s["case"]
    half, t = case["pairs"] == "half", s["q"].dtype
    valid = None
    if s["lens"] is not None:
        valid = (torch.arange(case["length"], device="cuda") < s["lens"][:, None]).view(*s["q"].shape[:-2], 1, 1)

    def rows(x):
        return x.float() if valid is None else torch.where(valid, x.float(), 0.0)

    res = {}
    for m in ("q", "k"):
        x, gamma = rows(s[m]), s["gamma_" + m]
        rstd = ((x * x).mean(-1, keepdim=True) + EPS) ** -0.5
        xhat = x * rstd
        res[m] = _turn(xhat * gamma.float(), cos, sin, half).to(t)
        if case["backward"]:
            g = _turn(rows(s["d" + m]), cos, -sin, half)
            # Sums over up to millions of rows: 64 bits.
            res["dgamma_" + m] = (g * xhat).flatten(0, -2).sum(0, dtype=torch.float64).to(gamma.dtype)
            g = g * gamma.float()
            res["d" + m] = (rstd * (g - xhat * (g * xhat).mean(-1, keepdim=True))).to(t)
    return res


def _codes(x, top, bits, mantissa):
    """8-bit codes of x (blocks of 256 with the largest magnitudes ``top``), uint8: magnitudes relative to ``top`` as
    floats of ``mantissa`` bits whose largest code is 1, the sign (7-bit magnitudes) above them. A magnitude rounds to the
    nearest, ties to even; below half the smallest it is 0 in a signed code, and the smallest in an unsigned one."""
    inv = torch.where(top >= torch.finfo(torch.float32).tiny, 1 / top, 0.0)
    r = (x.abs().view(-1, BLOCK) * inv[:, None]).view(-1)
    shift, high = 23 - mantissa, (1 << bits) - 1
    low = (127 << mantissa) - high  # what the shifted pattern of a float has above its code
    w = r.view(torch.int32)
    code = ((w + ((1 << (shift - 1)) - 1) + ((w >> shift) & 1)) >> shift) - low
    if bits == 7:
        least = _values(torch.ones(1, device="cuda", dtype=torch.uint8), 7, 3) * 0.5
        code = torch.where(r > least, code.clamp(1, high), 0)
        return torch.where(x < 0, code + 128, code).to(torch.uint8)
    return torch.where(r > 0, code.clamp(1, high), 0).to(torch.uint8)


def _values(code, bits, mantissa):
    """What codes stand for, relative to their block's largest magnitude."""
    c = code.int()
    c = c & 127 if bits == 7 else c
    high = (1 << bits) - 1
    v = ((c - high + (127 << mantissa)) << (23 - mantissa)).view(torch.float32)
    v = torch.where(c == 0, 0.0, v)
    return torch.where(code >= 128, -v, v) if bits == 7 else v


def _decoded(code, top, bits, mantissa):
    return (_values(code, bits, mantissa).view(-1, BLOCK) * top[:, None]).view(-1)


def _plain_adamw(s):
    b1, b2 = BETAS
    eight = s["scales"] is not None
    if eight:
        m = _decoded(s["m"], s["scales"][:, 0], 7, 3)
        u = _decoded(s["v"], s["scales"][:, 1], 8, 4)
        v = u * u
    else:
        m, v = s["m"], s["v"]
    g = s["flat_g"].float() * s["grad_scale"]
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    u = v.sqrt()
    denom = u * (1 / math.sqrt(1 - b2 ** s["step"])) + ADAM_EPS
    p = s["flat_p"].float() * (1 - LR * DECAY) - m / denom * (LR / (1 - b1 ** s["step"]))
    s["flat_p"].copy_(p)
    if not eight:
        s["m"].copy_(m)
        s["v"].copy_(v)
        return {"p": s["flat_p"], "m": s["m"], "v": s["v"]}
    top_m, top_u = (x.view(-1, BLOCK).abs().amax(1) for x in (m, u))
    s["m"].copy_(_codes(m, top_m, 7, 3))
    s["v"].copy_(_codes(u, top_u, 8, 4))
    s["scales"].copy_(torch.stack((top_m, top_u), 1))
    u = _decoded(s["v"], top_u, 8, 4)
    return {"p": s["flat_p"], "m": _decoded(s["m"], top_m, 7, 3), "v": u * u}


def _plain_grad_norm(s):
    # Sums over up to hundreds of millions of values: 64 bits.
    norm = s["flat_g"].float().square().sum(dtype=torch.float64).sqrt()
    return {"norm": norm.float(), "scale": torch.where(norm > 1.0, 1.0 / norm, 1.0).float()}


# ------------------------------------------------------------------------------- the framework's calls


def _own_rotary(s):
    from unblend_b200 import training

    args = (s["freqs"], s["positions"], s["case"]["pairs"] == "interleaved", s["scale"])
    q, k = training.rotary_forward(s["q"], s["k"], *args)
    if not s["case"]["backward"]:
        return {"q": q, "k": k}
    dq, dk = training.rotary_backward(s["dq"], s["dk"], *args)
    return {"q": q, "k": k, "dq": dq, "dk": dk}


def _own_qk_norm(s):
    from unblend_b200 import training

    args = (s["gamma_q"], s["gamma_k"], s["freqs"], s["positions"], s["case"]["pairs"] == "interleaved", s["scale"],
            EPS, s["lens"])
    q, k = training.qk_norm_rotary_forward(s["q"], s["k"], *args)
    if not s["case"]["backward"]:
        return {"q": q, "k": k}
    dq, dk, dgamma_q, dgamma_k = training.qk_norm_rotary_backward(s["dq"], s["dk"], s["q"], s["k"], *args)
    return {"q": q, "k": k, "dq": dq, "dk": dk, "dgamma_q": dgamma_q, "dgamma_k": dgamma_k}


def _own_adamw(s):
    from unblend_b200 import training

    moments = training.AdamWState(s["m"], s["v"], s["scales"])
    training.adamw_step(s["params"], s["grads"], moments, s["step"], LR, BETAS, ADAM_EPS, DECAY, s["grad_scale"])
    m, v = training.adamw_moments(moments)
    return {"p": s["flat_p"], "m": m, "v": v}


def _own_grad_norm(s):
    from unblend_b200 import training

    norm, scale = training.grad_norm(s["grads"], 1.0)
    return {"norm": norm, "scale": scale}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"rotary": _own_rotary, "qk_norm": _own_qk_norm, "adamw": _own_adamw,
                "grad_norm": _own_grad_norm}[op](state)
    return {"rotary": _plain_rotary, "qk_norm": _plain_qk_norm, "adamw": _plain_adamw,
            "grad_norm": _plain_grad_norm}[op](state)


# ----------------------------------------------------------------------------------------------- work


def work(case):
    if case["op"] in ("adamw", "grad_norm"):
        n = float(sum(math.prod(x) for x in _shapes(case)))
        if case["op"] == "grad_norm":
            return {"bytes": n * SIZE[case["grads"]], "flops": 2.0 * n}
        # Parameters and moments are read and written, gradients read; 8-bit moments are handed out as values too.
        moments = 16.0 if case["bits"] == 32 else 4.0 + 16.0 / BLOCK + 8.0
        return {"bytes": n * (2 * SIZE[case["dtype"]] + SIZE[case["grads"]] + moments), "flops": 15.0 * n}
    rows = float(case["outer"] * case["inner"] * case["length"] * (case["heads"] + case["kv_heads"]))
    n, e = rows * case["hd"], SIZE[case["dtype"]]
    share = 0.5 if case["ragged"] else 1.0  # lengths are uniform in [0, full]; rows behind them are only written
    if case["op"] == "rotary":
        return {"bytes": (4.0 if case["backward"] else 2.0) * n * e, "flops": (6.0 if case["backward"] else 3.0) * n}
    if not case["backward"]:
        return {"bytes": (1.0 + share) * n * e, "flops": 7.0 * n * share}
    return {"bytes": (2.0 + 3.0 * share) * n * e, "flops": 21.0 * n * share}


# --------------------------------------------------------------------------------------------- 64 bits


def _phases(s):
    """exp(i angle) times the factor, complex, [..., length, 1, n]."""
    n = s["case"]["length"]
    p = torch.arange(n, device="cuda", dtype=torch.float64) if s["positions"] is None else s["positions"].double()
    z = torch.einsum("...l,n->...ln", p, s["freqs"]).unsqueeze(-2)
    return torch.polar(torch.full_like(z, s["scale"]), z)


def _exact_turn(x, phase, half):
    n = phase.shape[-1]
    x, rest = x[..., :2 * n], x[..., 2 * n:]
    pair = x.unflatten(-1, (2, n)).transpose(-1, -2) if half else x.unflatten(-1, (n, 2))
    z = torch.view_as_real(torch.complex(pair[..., 0], pair[..., 1]) * phase)
    return torch.cat(((z.transpose(-1, -2) if half else z).flatten(-2), rest), -1)


def _exact_rotary(s):
    phase, half = _phases(s), s["case"]["pairs"] == "half"
    got = {}
    for m in ("q", "k"):
        got[m] = _exact_turn(s[m].double(), phase, half)
        if s["case"]["backward"]:
            got["d" + m] = _exact_turn(s["d" + m].double(), phase.conj(), half)
    return got


def _exact_qk_norm(s):
    """A slice of the sequences' heads at a time, gradients by differentiation of the definition."""
    case = s["case"]
    phase, half = _phases(s), case["pairs"] == "half"
    got = {}
    for m in ("q", "k"):
        full = s[m]
        out, din = torch.empty(full.shape, dtype=torch.float64, device="cuda"), None
        gamma = s["gamma_" + m].double().requires_grad_()
        dgamma = torch.zeros_like(gamma)
        if case["backward"]:
            din = torch.empty_like(out)
        for h in range(full.shape[-2]):
            x = full[..., h, :].double()
            dy = s["d" + m][..., h, :].double() if case["backward"] else None
            if s["lens"] is not None:
                inside = (torch.arange(case["length"], device="cuda")[None] < s["lens"][:, None])[..., None]
                x = torch.where(inside, x, 0.0)
                dy = None if dy is None else torch.where(inside, dy, 0.0)
            x.requires_grad_()
            y = _exact_turn(x / (x.pow(2).mean(-1, keepdim=True) + EPS).sqrt() * gamma, phase[..., 0, :], half)
            out[..., h, :] = y.detach()
            if case["backward"]:
                dx, dg = torch.autograd.grad(y, (x, gamma), dy)
                din[..., h, :] = dx
                dgamma = dgamma + dg
        got[m] = out
        if case["backward"]:
            got["d" + m], got["dgamma_" + m] = din, dgamma.detach()
    return got


def _exact_adamw(s):
    """The parameters, and moments of 32 bits; what 8 bits hold next to a border of two codes has no such value."""
    (b1, b2), t = BETAS, s["step"]
    if s["scales"] is None:
        m, v = s["m"].double(), s["v"].double()
    else:
        # Signed codes: 2^((c - 127) / 8) with a linear mantissa; unsigned: the same with 16 steps an octave.
        c = torch.arange(128, device="cuda", dtype=torch.float64) - 127
        mag = (1 + (c - 8 * (c / 8).floor()) / 8) * 2.0 ** (c / 8).floor()
        mag[0] = 0
        tab_m = torch.cat((mag, -mag))
        c = torch.arange(256, device="cuda", dtype=torch.float64) - 255
        tab_u = (1 + (c - 16 * (c / 16).floor()) / 16) * 2.0 ** (c / 16).floor()
        tab_u[0] = 0
        top = s["scales"].double().repeat_interleave(BLOCK, 0)
        m, v = tab_m[s["m"].long()] * top[:, 0], (tab_u[s["v"].long()] * top[:, 1]) ** 2
    g, p = s["flat_g"].double() * s["grad_scale"].double(), s["flat_p"].double()
    m, v = torch.lerp(g, m, b1), torch.lerp(g.square(), v, b2)
    step = (m / (1 - b1**t)) / ((v / (1 - b2**t)).sqrt() + ADAM_EPS)
    p = p - LR * (step + DECAY * p)
    return {"p": p, "m": m, "v": v} if s["scales"] is None else {"p": p, "m": None, "v": None}


def _exact_grad_norm(s):
    norm = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(x.double()) for x in s["grads"]]))
    return {"norm": norm, "scale": 1.0 / norm.clamp(min=1.0)}


def exact(case, seed):
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "qk_norm": _exact_qk_norm, "adamw": _exact_adamw,
            "grad_norm": _exact_grad_norm}[case["op"]](s)
