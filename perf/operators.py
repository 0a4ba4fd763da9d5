"""The training operators of ``unblend_b200.training`` as measured calls: layer norm, attention and dropout-add,
each with its backward pass, at the sizes that fine-tuning and running the separation transformers give them.

``run`` takes one pass through an operator: in elementary torch operations where ``own`` is false, through the
framework's public functions where it is true. ``exact`` gives the same outputs from the definition in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-5


# ---------------------------------------------------------------------------------------------- cases


def _norm(name, outer, rows, cols, dtype, weights="fp32", pad=0):
    """``pad``: columns of the buffer behind each row that the norm does not see."""
    return {"name": name, "op": "layer_norm", "outer": outer, "rows": rows, "cols": cols, "dtype": dtype,
            "weights": weights, "pad": pad}


def _attn(name, outer, inner, lq, lk, heads, kv_heads, hd, dtype, layout="split", causal=False, ragged=False,
          backward=True):
    """``layout``: "split" q, k, v of their own; "packed" column blocks of one projection; "axis" packed, with the
    sequences running along the first of two token axes; "ragged": per-sequence lengths in a padded batch."""
    return {"name": name, "op": "attention", "outer": outer, "inner": inner, "lq": lq, "lk": lk, "heads": heads,
            "kv_heads": kv_heads, "hd": hd, "dtype": dtype, "layout": layout, "causal": causal, "ragged": ragged,
            "backward": backward}


def _drop(name, rows, cols, dtype, stream, p, scale):
    """``stream``: type of the residual stream that the dropped branch is added to."""
    return {"name": name, "op": "dropout_add", "rows": rows, "cols": cols, "dtype": dtype, "stream": stream, "p": p,
            "scale": scale}


def listed():
    return [
        # One STFT frame of a 62-band separator: the smallest call, where launches count.
        _norm("norm one frame", 1, 62, 512, "fp32"),
        # Odd width, rows that are a slice of wider ones: 16-bit, with weights of the same type.
        _norm("norm odd slice", 3, 1111, 5003, "fp16", "fp16", pad=6),
        # Many tokens of a wide model, bf16 activations and fp32 weights: bandwidth alone.
        _norm("norm many wide tokens", 1, 262147, 1024, "bf16"),
        # fp32 training of a short clip: the smallest attention call.
        _attn("attention short clip fp32", 2, 1, 161, 161, 8, 8, 64, "fp32"),
        # Band axis of an axial model: 801 sequences of 62 tokens out of one packed projection.
        _attn("attention band axis", 1, 801, 62, 62, 8, 8, 64, "bf16", layout="packed"),
        # Time axis of the same tokens: 62 sequences of 801, rows far apart in memory.
        _attn("attention time axis", 1, 62, 801, 801, 8, 8, 64, "bf16", layout="axis"),
        # Cross attention between the branches: 2688 frequency tokens read 1344 time tokens.
        _attn("attention cross branch", 8, 1, 2688, 1344, 8, 8, 64, "bf16"),
        # Padded batch of clips with their own lengths (some empty), 48-wide heads.
        _attn("attention padded fp16", 6, 1, 1000, 1343, 8, 8, 48, "fp16", ragged=True),
        # Long causal sequence with shared key/value heads.
        _attn("attention long causal", 1, 1, 8192, 8192, 16, 4, 128, "bf16", causal=True),
        # One new token per stream over a long context: the serving call, forward alone.
        _attn("attention one token", 4, 1, 1, 8191, 16, 4, 128, "bf16", ragged=True, backward=False),
        # Residual update behind an attention block: bf16 branch into the fp32 stream, with LayerScale.
        _drop("dropout block residual", 86016, 512, "bf16", "fp32", 0.1, True),
        # The same for the few tokens of one clip, fp32: launches count.
        _drop("dropout one clip", 336, 512, "fp32", "fp32", 0.2, True),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["layer_norm", "attention", "attention", "attention", "dropout_add"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op == "layer_norm":
        cols = log(32, 8192)
        rows = log(16, max(17, min(262144, (1 << 27) // cols)))
        c = _norm("", 1, rows, cols, dtype, rng.choice(["fp32", dtype]), rng.choice([0, 0, 8, 3]))
    elif op == "dropout_add":
        cols = log(32, 4096)
        rows = log(16, max(17, min(262144, (1 << 25) // cols)))
        c = _drop("", rows, cols, dtype, rng.choice(["fp32", dtype]), rng.choice([0.05, 0.1, 0.25, 0.5]),
                  rng.random() < 0.7)
    else:
        heads = rng.choice([4, 8, 12, 16])
        hd = rng.choice([32, 48, 64, 64, 80, 96, 128, 128])
        lq, lk = log(1, 8192), log(16, 8192)
        if rng.random() < 0.5:
            lk = max(16, lq)
        lq = min(lq, lk) if rng.random() < 0.5 else lq
        cap = (1 << 29) if dtype == "fp32" else (1 << 33)  # score entries x head width
        outer = max(1, min(log(1, 512), cap // (heads * lq * lk * hd)))
        while heads * lq * lk * hd * outer > cap:
            lq, lk = max(1, lq // 2), max(16, lk // 2)
        layout = rng.choice(["split", "split", "packed", "axis"])
        if layout != "split":
            lk = lq = max(lq, 2)
            while heads * lq * lk * hd * outer > cap:
                lq = lk = lq // 2
        kv = heads if layout != "split" else rng.choice([heads, heads // 2, heads // 4])
        c = _attn("", 1 if layout == "axis" else outer, outer if layout == "axis" else 1, lq, lk, heads, kv, hd,
                  dtype, layout, rng.random() < 0.4, rng.random() < 0.3 and layout != "axis",
                  rng.random() < 0.8)
    del c["name"]
    return c


# --------------------------------------------------------------------------------------------- inputs


def _rows_of(case, g, dtype, mean=0.0):
    """[outer, rows, cols] values inside rows of cols + pad."""
    x = torch.randn(case["outer"], case["rows"], case["cols"] + case["pad"], device="cuda", generator=g)
    return (x * 1.5 + mean).to(dtype)[..., : case["cols"]]


def _prepare_norm(case, g):
    t, tw = DTYPES[case["dtype"]], DTYPES[case["weights"]]
    cols = case["cols"]
    return {"x": _rows_of(case, g, t, 0.3), "dy": _rows_of(case, g, t),
            "gamma": (1 + 0.2 * torch.randn(cols, device="cuda", generator=g)).to(tw),
            "beta": (0.1 * torch.randn(cols, device="cuda", generator=g)).to(tw)}


def _prepare_attn(case, g):
    t = DTYPES[case["dtype"]]
    o, i, lq, lk, h, hk, hd = (case[n] for n in ("outer", "inner", "lq", "lk", "heads", "kv_heads", "hd"))

    def rand(*shape):
        return torch.randn(*shape, device="cuda", generator=g).to(t)

    if case["layout"] == "split":
        q, k, v = rand(o * i, lq, h, hd), rand(o * i, lk, hk, hd), rand(o * i, lk, hk, hd)
        dout = rand(o * i, lq, h, hd)
    elif case["layout"] == "packed":
        q, k, v = rand(o * i, lq, 3, h, hd).unbind(2)
        dout = rand(o * i, lq, h, hd)
    else:  # tokens are [outer, sequence position, inner]: the sequences of (outer, inner) run along the middle
        q, k, v = (x.transpose(1, 2) for x in rand(o, lq, i, 3, h, hd).unbind(3))
        dout = rand(o, lq, i, h, hd).transpose(1, 2)
    s = {"q": q, "k": k, "v": v, "dout": dout, "q_lens": None, "k_lens": None}
    if case["ragged"]:
        n = o * i
        s["k_lens"] = torch.randint(0, lk + 1, (n,), device="cuda", generator=g, dtype=torch.int32)
        if case["backward"]:
            s["q_lens"] = torch.randint(0, lq + 1, (n,), device="cuda", generator=g, dtype=torch.int32)
    return s


def _prepare_drop(case, g):
    t, ts = DTYPES[case["dtype"]], DTYPES[case["stream"]]
    shape = (case["rows"], case["cols"])
    return {"x": torch.randn(shape, device="cuda", generator=g).to(t),
            "residual": torch.randn(shape, device="cuda", generator=g).to(ts),
            "dy": torch.randn(shape, device="cuda", generator=g).to(ts),
            "scale": 0.1 * torch.randn(case["cols"], device="cuda", generator=g) if case["scale"] else None,
            # (seed, offset) of the random numbers
            "rng": torch.randint(0, 1 << 40, (2,), device="cuda", generator=g)}


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    make = {"layer_norm": _prepare_norm, "attention": _prepare_attn, "dropout_add": _prepare_drop}[case["op"]]
    return {"case": dict(case), **make(case, g)}


# ---------------------------------------------------------------------------------------- plain forms


def _plain_norm(s):
    x, dy, gamma = s["x"].float(), s["dy"].float(), s["gamma"].float()
    xc = x - x.mean(-1, keepdim=True)
    rstd = ((xc * xc).mean(-1, keepdim=True) + EPS) ** -0.5
    xhat = xc * rstd
    y = xhat * gamma + s["beta"].float()
    gy = dy * gamma
    dx = rstd * (gy - gy.mean(-1, keepdim=True) - xhat * (gy * xhat).mean(-1, keepdim=True))
    t, tw = s["x"].dtype, s["gamma"].dtype
    # Sums over up to hundreds of thousands of rows: 64 bits.
    dgamma = (dy * xhat).sum((0, 1), dtype=torch.float64)
    dbeta = dy.sum((0, 1), dtype=torch.float64)
    return {"y": y.to(t), "dx": dx.to(t), "dgamma": dgamma.to(tw), "dbeta": dbeta.to(tw)}


def _visible(s):
    """[n, lq, lk] (or broadcastable) truth values: which key each query sees; and the valid rows of q and k."""
    case = s["case"]
    n, lq, lk = case["outer"] * case["inner"], case["lq"], case["lk"]
    ql = torch.full((n,), lq, device="cuda") if s["q_lens"] is None else s["q_lens"].long()
    kl = torch.full((n,), lk, device="cuda") if s["k_lens"] is None else s["k_lens"].long()
    i = torch.arange(lq, device="cuda")[None, :, None]
    j = torch.arange(lk, device="cuda")[None, None, :]
    see = (i < ql[:, None, None]) & (j < kl[:, None, None])
    if case["causal"]:
        see = see & (j <= i + (kl - ql)[:, None, None])
    return see


def _plain_attn(s):
    case = s["case"]
    t, rep, hd = s["q"].dtype, case["heads"] // case["kv_heads"], case["hd"]
    masked = case["causal"] or case["ragged"]

    def heads_first(x, rep=1):  # -> [n, heads, length, hd], 32 bits
        x = x.reshape(-1, *x.shape[-3:]).transpose(1, 2).float()
        return x.repeat_interleave(rep, 1) if rep > 1 else x

    def tokens_first(x, like):  # -> the layout of the call, rounded
        return x.transpose(1, 2).reshape(*like.shape).to(t)

    q, k, v = heads_first(s["q"]), heads_first(s["k"], rep), heads_first(s["v"], rep)
    scale = hd ** -0.5
    score = (q @ k.transpose(-1, -2)) * scale
    if masked:
        see = _visible(s)[:, None]
        score = score.masked_fill(~see, -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = (score - top).exp()
    del score
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    out = p @ v
    res = {"out": tokens_first(out, s["q"])}
    if not case["backward"]:
        return res
    dout = heads_first(s["dout"])

    def shared(x):  # sum over the query heads that share a key/value head
        return x.unflatten(1, (-1, rep)).sum(2) if rep > 1 else x

    res["dv"] = tokens_first(shared(p.transpose(-1, -2) @ dout), s["v"])
    ds = dout @ v.transpose(-1, -2)
    ds = p * (ds - (dout * out).sum(-1, keepdim=True)) * scale
    res["dq"] = tokens_first(ds @ k, s["q"])
    res["dk"] = tokens_first(shared(ds.transpose(-1, -2) @ q), s["k"])
    return res


def _philox_words(rng, n):
    """The first n 32-bit words of Philox-4x32-10 (Salmon et al., 2011): key = seed, counter = (index, offset)."""
    low = 0xFFFFFFFF
    blocks = torch.arange((n + 3) // 4, device="cuda")
    k0, k1 = rng[0] & low, (rng[0] >> 32) & low
    c0, c1 = blocks & low, blocks >> 32
    c2, c3 = rng[1] & low, (rng[1] >> 32) & low
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # wrapped 64-bit products: all bits are kept
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    c0, c1, c2, c3 = (torch.broadcast_to(c, blocks.shape) for c in (c0, c1, c2, c3))
    return torch.stack((c0, c1, c2, c3), 1).reshape(-1)[:n]


def _plain_drop(s):
    x, dy, p = s["x"].float(), s["dy"].float(), s["case"]["p"]
    keep = (_philox_words(s["rng"], x.numel()) >= round(p * 2.0**32)).view(x.shape)
    kept = torch.where(keep, x / (1 - p), 0.0)
    dkept = torch.where(keep, dy / (1 - p), 0.0)
    t, ts = s["x"].dtype, s["residual"].dtype
    if s["scale"] is None:
        return {"y": (s["residual"].float() + kept).to(ts), "dx": dkept.to(t)}
    return {"y": (s["residual"].float() + s["scale"] * kept).to(ts), "dx": (s["scale"] * dkept).to(t),
            "dscale": (dkept * x).sum(0, dtype=torch.float64).to(s["scale"].dtype)}


# ------------------------------------------------------------------------------- the framework's calls


def _own_norm(s):
    from unblend_b200 import training

    y, stats = training.layer_norm_forward(s["x"], s["gamma"], s["beta"], EPS)
    dx, dgamma, dbeta = training.layer_norm_backward(s["dy"], s["x"], stats, s["gamma"])
    return {"y": y, "dx": dx, "dgamma": dgamma, "dbeta": dbeta}


def _own_attn(s):
    from unblend_b200 import training

    kw = {"causal": s["case"]["causal"], "q_lens": s["q_lens"], "k_lens": s["k_lens"]}
    out, lse = training.attention_forward(s["q"], s["k"], s["v"], **kw)
    if not s["case"]["backward"]:
        return {"out": out}
    dq, dk, dv = training.attention_backward(s["dout"], s["q"], s["k"], s["v"], out, lse, **kw)
    return {"out": out, "dq": dq, "dk": dk, "dv": dv}


def _own_drop(s):
    from unblend_b200 import training

    p, rng = s["case"]["p"], s["rng"]
    y = training.dropout_add_forward(s["x"], p, rng, s["residual"], s["scale"])
    dx, dscale = training.dropout_add_backward(s["dy"], s["x"], p, rng, s["scale"])
    return {"y": y, "dx": dx} if dscale is None else {"y": y, "dx": dx, "dscale": dscale}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"layer_norm": _own_norm, "attention": _own_attn, "dropout_add": _own_drop}[op](state)
    return {"layer_norm": _plain_norm, "attention": _plain_attn, "dropout_add": _plain_drop}[op](state)


# ----------------------------------------------------------------------------------------------- work


def work(case):
    size = {"fp32": 4, "bf16": 2, "fp16": 2}
    e = size[case["dtype"]]
    if case["op"] == "layer_norm":
        n = case["outer"] * case["rows"] * case["cols"]
        # Forward reads x and writes y, backward reads dy and x and writes dx; gamma, beta and their gradients.
        return {"bytes": 5.0 * n * e + 5.0 * case["cols"] * size[case["weights"]], "flops": 20.0 * n}
    if case["op"] == "dropout_add":
        n, r = case["rows"] * case["cols"], size[case["stream"]]
        # Forward reads x and the residual and writes y, backward reads dy (and x for the scale) and writes dx.
        return {"bytes": float(n) * (2 * e + 3 * r + (e if case["scale"] else 0)), "flops": 40.0 * n}
    seqs, lq, lk, h, hk, hd = case["outer"] * case["inner"], case["lq"], case["lk"], case["heads"], \
        case["kv_heads"], case["hd"]
    pairs = float(lq) * lk
    if case["causal"]:  # query i of lq sees the first lk - lq + i + 1 keys
        m = min(lq, lk)
        pairs = m * (lk - (m - 1) / 2.0)
    share_q = 0.5 if case["ragged"] and case["backward"] else 1.0  # lengths are uniform in [0, full]
    share_k = 0.5 if case["ragged"] else 1.0
    nq, nk = seqs * lq * h * hd * e, seqs * lk * hk * hd * e
    if not case["backward"]:
        return {"bytes": nq * (1 + share_q) + 2 * nk * share_k, "flops": 4.0 * seqs * h * hd * pairs * share_k}
    # Inputs q, k, v, dout are read up to the lengths; out, dq, dk, dv are written whole.
    return {"bytes": 2 * nq * (1 + share_q) + 2 * nk * (1 + share_k),
            "flops": 14.0 * seqs * h * hd * pairs * share_q * share_k}


# --------------------------------------------------------------------------------------------- 64 bits


def _exact_norm(s):
    x = s["x"].double().requires_grad_()
    gamma, beta = s["gamma"].double().requires_grad_(), s["beta"].double().requires_grad_()
    var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
    y = (x - mean) / (var + EPS).sqrt() * gamma + beta
    dx, dgamma, dbeta = torch.autograd.grad(y, (x, gamma, beta), s["dy"].double())
    return {"y": y.detach(), "dx": dx, "dgamma": dgamma, "dbeta": dbeta}


def _exact_attn(s):
    """One sequence and key/value head at a time, cut to its lengths; gradients by differentiation of the definition."""
    case = s["case"]
    rep, hd, lq, lk = case["heads"] // case["kv_heads"], case["hd"], case["lq"], case["lk"]
    flat = {n: s[n].reshape(-1, *s[n].shape[-3:]) for n in ("q", "k", "v", "dout")}
    n = flat["q"].shape[0]
    many = n if not case["ragged"] else 1  # equal lengths: all sequences of a head at once
    got = {m: torch.zeros(flat[f].shape, dtype=torch.float64, device="cuda")
           for m, f in (("out", "q"), ("dq", "q"), ("dk", "k"), ("dv", "v"))}
    for b in range(0, n, many):
        ql = lq if s["q_lens"] is None else int(s["q_lens"][b])
        kl = lk if s["k_lens"] is None else int(s["k_lens"][b])
        first = max(0, ql - kl) if case["causal"] else 0  # queries before it see no key
        if kl == 0 or first >= ql:
            continue
        for h in range(case["kv_heads"]):
            at = slice(b, b + many)
            k = flat["k"][at, :kl, h].double().requires_grad_()
            v = flat["v"][at, :kl, h].double().requires_grad_()
            for r in range(h * rep, (h + 1) * rep):
                q = flat["q"][at, first:ql, r].double().requires_grad_()
                z = torch.einsum("bid,bjd->bij", q, k) / math.sqrt(hd)
                if case["causal"]:
                    late = torch.ones(ql - first, kl, dtype=torch.bool, device="cuda").triu(kl - ql + first + 1)
                    z = z.masked_fill(late, -math.inf)
                y = torch.einsum("bij,bjd->bid", z.softmax(-1), v)
                got["out"][at, first:ql, r] = y.detach()
                if case["backward"]:
                    dq, dk, dv = torch.autograd.grad(y, (q, k, v), flat["dout"][at, first:ql, r].double())
                    got["dq"][at, first:ql, r] = dq
                    got["dk"][at, :kl, h] += dk
                    got["dv"][at, :kl, h] += dv
    names = {"out": "q", "dq": "q", "dk": "k", "dv": "v"} if case["backward"] else {"out": "q"}
    return {m: got[m].view(s[f].shape) for m, f in names.items()}


def _exact_drop(s):
    seed, offset = (int(x) for x in s["rng"].tolist())
    n, p = s["x"].numel(), s["case"]["p"]
    block = torch.arange((n + 3) // 4, device="cuda")

    def times(x, m):
        """High and low word of x * m by 16-bit limbs."""
        xl, xh, ml, mh = x & 0xFFFF, x >> 16, m & 0xFFFF, m >> 16
        mid = xh * ml + ((xl * ml) >> 16)
        cross = xl * mh + (mid & 0xFFFF)
        return xh * mh + (mid >> 16) + (cross >> 16), ((cross & 0xFFFF) << 16) | ((xl * ml) & 0xFFFF)

    ctr = [block % 2**32, block // 2**32, torch.full_like(block, offset % 2**32),
           torch.full_like(block, offset // 2**32 % 2**32)]
    key = [seed % 2**32, seed // 2**32 % 2**32]
    for _ in range(10):
        (h0, l0), (h1, l1) = times(ctr[0], 0xD2511F53), times(ctr[2], 0xCD9E8D57)
        ctr = [h1 ^ ctr[1] ^ key[0], l1, h0 ^ ctr[3] ^ key[1], l0]
        key = [(key[0] + 0x9E3779B9) % 2**32, (key[1] + 0xBB67AE85) % 2**32]
    word = torch.stack(ctr, -1).flatten()[:n].view(s["x"].shape)
    mask = (word >= round(p * 2.0**32)).double() / (1 - p)
    x, dy = s["x"].double(), s["dy"].double()
    scale = torch.ones(x.shape[1], device="cuda", dtype=torch.float64) if s["scale"] is None else s["scale"].double()
    got = {"y": s["residual"].double() + scale * mask * x, "dx": scale * mask * dy}
    if s["scale"] is not None:
        got["dscale"] = (mask * x * dy).sum(0)
    return got


def exact(case, seed):
    s = prepare(case, seed)
    return {"layer_norm": _exact_norm, "attention": _exact_attn, "dropout_add": _exact_drop}[case["op"]](s)
