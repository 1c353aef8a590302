"""Cases for the 8-bit activation checkpoints and the residual norms of vita_amd.

Format of a checkpoint (what the plain forms below compute with elementary operations): a row is cut into groups of 32
neighbours, each group has a power-of-two scale 2^e, e the smallest integer in [-117, 119] with amax / 2^e <= 448 (amax over the
group's finite values), and each value is stored as the e4m3 number next to value / 2^e (ties to even, clamped to +-448; NaN and
infinities as NaN).  A scale is kept as the byte e + 127.  A stored value code * 2^e is exact in bf16, so that is the type in
which the stored values are returned.
"""
import math

import torch

own = False

GROUP = 32
BF16, F32 = torch.bfloat16, torch.float32
TYPES = {"bf16": BF16, "f32": F32}


# ------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one token of a serving loop: bf16 stream, the normalised row only in 8 bits (latency)
        {"name": "norm fwd, 1 row", "op": "norm_fwd", "rows": 1, "d": 1025, "kind": "rms", "x": "bf16", "res": "bf16",
         "y": False, "pack": "output"},
        # decoder layer at T = 50, two subjects: fp32 residual stream, bf16 branch, y for the product and n as its checkpoint
        {"name": "norm fwd, 46082 rows", "op": "norm_fwd", "rows": 46082, "d": 1025, "kind": "rms", "x": "bf16", "res": "f32",
         "y": True, "pack": "normed"},
        # norm1 / norm2 of an encoder layer at T = 50: LayerNorm gradient from the 8-bit rows, residual gradient joined
        {"name": "norm bwd, 13826 rows", "op": "norm_bwd", "rows": 13826, "d": 1025, "kind": "layer", "src": "act8", "dy": "bf16",
         "dx": "f32", "dx_in": True},
        # the same operator over a bf16 stream that was kept whole, wider rows
        {"name": "norm bwd, 4096 x 4096", "op": "norm_bwd", "rows": 4096, "d": 4096, "kind": "rms", "src": "bf16", "dy": "bf16",
         "dx": "bf16", "dx_in": True},
        # MLP of the tabular tower: 32 subjects x 118 tokens
        {"name": "gelu fwd, 3776 rows", "op": "gelu_fwd", "rows": 3776, "d": 4100},
        # MLP of an encoder layer at T = 50
        {"name": "gelu fwd, 13826 rows", "op": "gelu_fwd", "rows": 13826, "d": 4100},
        {"name": "gelu bwd, 3776 rows", "op": "gelu_bwd", "rows": 3776, "d": 4100},
        # MLP of a decoder layer at T = 50 (the largest tensors of the step)
        {"name": "gelu bwd, 46082 rows", "op": "gelu_bwd", "rows": 46082, "d": 4100},
        # weight gradients of the first MLP product (tabular tower) and of q, k, v (encoder layer)
        {"name": "wgrad, 3776 tokens", "op": "wgrad", "rows": 3776, "d": 1025, "m": 4100},
        {"name": "wgrad, 13826 tokens", "op": "wgrad", "rows": 13826, "d": 1025, "m": 3075},
        # the input of the decoder's embedding: packed in the forward pass ...
        {"name": "pack, 13826 rows", "op": "pack", "rows": 13826, "d": 1025, "x": "f32"},
        # ... and a norm's output restored for the weight gradient behind it
        {"name": "restore, 13826 rows", "op": "restore", "rows": 13826, "d": 1025, "affine": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm_fwd", "norm_bwd", "gelu_fwd", "gelu_bwd", "wgrad", "pack", "restore"])
    # a norm's gradient over 1 or 2 columns is a difference of equal numbers: what is left of it is rounding on every side
    d = _log_int(rng, 8 if op == "norm_bwd" else 1, 8192)
    rows = min(_log_int(rng, 1, 46082), max(1, 46082 * 1025 // d))
    c = {"op": op, "rows": rows, "d": d}
    if op == "norm_fwd":
        pack = rng.choice(["none", "normed", "output"])
        c.update(kind=rng.choice(["rms", "layer"]), x=rng.choice(["bf16", "f32"]), res=rng.choice(["none", "bf16", "f32"]),
                 y=pack == "none" or rng.random() < 0.7, pack=pack)
    elif op == "norm_bwd":
        c.update(kind=rng.choice(["rms", "layer"]), src=rng.choice(["act8", "bf16", "f32"]), dy=rng.choice(["bf16", "f32"]),
                 dx=rng.choice(["bf16", "f32"]), dx_in=rng.random() < 0.5)
    elif op == "wgrad":
        c["d"], c["m"] = _log_int(rng, 8, 4100), _log_int(rng, 8, 4100)
        c["rows"] = min(_log_int(rng, 1, 46082), max(1, 46082 * 1025 * 1025 // (c["d"] * c["m"])))
    elif op == "pack":
        c["x"] = rng.choice(["bf16", "f32"])
    elif op == "restore":
        c["affine"] = rng.random() < 0.5
    return c


def work(case):
    op, r, d = case["op"], case["rows"], case["d"]
    n, size = r * d, {"bf16": 2, "f32": 4, "none": 0, False: 0, True: 2}
    act, values = n + r * -(-d // GROUP), 2 * n          # codes and scales; the values that they stand for
    if op == "norm_fwd":
        stream = max(size[case["x"]], size[case["res"]]) if case["res"] != "none" else 0
        b = n * (size[case["x"]] + size[case["res"]] + stream + size[case["y"]]) + 8 * d + 4 * r
        return {"bytes": b + (act + values if case["pack"] != "none" else 0), "flops": 8 * n}
    if op == "norm_bwd":
        src = act if case["src"] == "act8" else n * size[case["src"]]
        return {"bytes": src + n * (size[case["dy"]] + size[case["dx"]] * (2 if case["dx_in"] else 1)) + 12 * d + 4 * r, "flops": 12 * n}
    if op == "gelu_fwd":
        return {"bytes": 4 * n + act + values, "flops": 20 * n}
    if op == "gelu_bwd":
        return {"bytes": 6 * n + act, "flops": 25 * n}
    if op == "wgrad":
        return {"bytes": act + 2 * r * case["m"] + 4 * case["m"] * d, "flops": 2.0 * n * case["m"]}
    if op == "pack":
        return {"bytes": n * size[case["x"]] + act + values, "flops": 4 * n}
    return {"bytes": act + values + (8 * d if case["affine"] else 0), "flops": 3 * n}


# ------------------------------------------------------------------------------------------------------------ inputs
def _rows(rows, d, dtype, scale, gen, step=8):
    """[rows, d] on rows of a multiple of `step` elements, as the framework lays out its streams (pads are zero)."""
    t = torch.zeros(rows, -(-d // step) * step, dtype=dtype, device="cuda")
    t[:, :d] = (torch.randn(rows, d, device="cuda", generator=gen) * scale).to(dtype)
    return t[:, :d]


def _codes(rows, d, scale, gen):
    """A checkpoint in hand before the call: e4m3 codes [rows, 32 n] and their scale bytes [rows, n]."""
    n = -(-d // GROUP)
    v = torch.zeros(rows, n * GROUP, device="cuda")
    v[:, :d] = torch.randn(rows, d, device="cuda", generator=gen) * scale
    e = _exponents(v.view(rows, n, GROUP))
    q = (v.view(rows, n, GROUP) * torch.exp2(-e.float()).unsqueeze(-1)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return q.view(rows, n * GROUP), (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, r, d = case["op"], case["rows"], case["d"]
    s = {"case": case, "d": d}
    if op in ("norm_fwd", "norm_bwd", "restore"):
        s["gamma"] = 1 + 0.1 * torch.randn(d, device="cuda", generator=gen)
        s["beta"] = 0.1 * torch.randn(d, device="cuda", generator=gen)
        if case.get("kind") == "rms" or not case.get("affine", True):
            s["beta"] = None
        if not case.get("affine", True):
            s["gamma"] = None
    if op == "norm_fwd":
        s["eps"] = 1e-6 if case["kind"] == "rms" else 1e-5
        s["x"] = _rows(r, d, TYPES[case["x"]], 0.5, gen, 64)
        s["res"] = _rows(r, d, TYPES[case["res"]], 2.0, gen, 64) if case["res"] != "none" else None
    elif op == "norm_bwd":
        if case["src"] == "act8":
            s["q"], s["scale"] = _codes(r, d, 1.0, gen)
            s["rstd"] = 0.3 + torch.rand(r, device="cuda", generator=gen)
            s["mean"] = None
        else:
            s["sum"] = _rows(r, d, TYPES[case["src"]], 2.0, gen, 64)
            x = s["sum"].double()
            mean = x.mean(1, keepdim=True) if case["kind"] == "layer" else torch.zeros_like(x[:, :1])
            s["rstd"] = torch.rsqrt((x - mean).square().mean(1) + 1e-5).float()
            s["mean"] = mean[:, 0].float() if case["kind"] == "layer" else None
        s["dy"] = _rows(r, d, TYPES[case["dy"]], 1e-3, gen, 64)
        s["dx_in"] = _rows(r, d, TYPES[case["dx"]], 1e-3, gen, 64) if case["dx_in"] else None
    elif op == "gelu_fwd":
        s["z"] = _rows(r, d, BF16, 1.2, gen, 64)
    elif op in ("gelu_bwd", "restore"):
        s["q"], s["scale"] = _codes(r, d, 1.2, gen)
        if op == "gelu_bwd":
            s["dg"] = _rows(r, d, BF16, 1e-3, gen, 64)
    elif op == "wgrad":
        s["q"], s["scale"] = _codes(r, d, 1.0, gen)
        s["dy"] = _rows(r, case["m"], BF16, 1e-3, gen)
    elif op == "pack":
        s["x"] = _rows(r, d, TYPES[case["x"]], 1.0, gen, 64)
    return s


# ------------------------------------------------------------------------------------------------------------ plain forms
def _exponents(g):
    """The scale exponents of groups [..., GROUP]; in 64 bits, as amax / 448 may lie next to a power of two."""
    a = g.abs().double()
    amax = torch.where(torch.isfinite(a), a, torch.zeros_like(a)).amax(-1)
    m, e = torch.frexp(amax / 448.0)
    return torch.where(amax > 0, e - (m == 0.5).to(e.dtype), torch.full_like(e, -117)).clamp(-117, 119)


def _stored(x):
    """The values that the checkpoint of fp32 rows [rows, d] stands for, in bf16."""
    r, d = x.shape
    n = -(-d // GROUP)
    g = torch.zeros(r, n * GROUP, device=x.device)
    g[:, :d] = x
    g = g.view(r, n, GROUP)
    s = torch.exp2(_exponents(g).float()).unsqueeze(-1)
    v = torch.where(torch.isfinite(g), (g / s).clamp(-448.0, 448.0), torch.full_like(g, math.nan))
    return (v.to(torch.float8_e4m3fn).float() * s).view(r, n * GROUP)[:, :d].to(BF16)


def _values(s):
    q = s["q"].float()
    e = s["scale"].view(torch.uint8).float() - 127.0
    return (q.view(q.shape[0], -1, GROUP) * torch.exp2(e).unsqueeze(-1)).view(q.shape)[:, :s["d"]]


def _cdf(z):
    return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5)))


def _run_plain(s):
    case = s["case"]
    op = case["op"]
    if op == "norm_fwd":
        t = s["x"].float()
        out = {}
        if s["res"] is not None:
            t = t + s["res"].float()
            out["sum"] = t.to(F32 if F32 in (s["x"].dtype, s["res"].dtype) else BF16)
        c = t - t.mean(1, keepdim=True) if case["kind"] == "layer" else t
        rstd = torch.rsqrt(c.square().mean(1, keepdim=True) + s["eps"])
        n = c * rstd
        y = n * s["gamma"] if s["beta"] is None else n * s["gamma"] + s["beta"]
        out["rstd"] = rstd[:, 0]
        if case["y"]:
            out["y"] = y.to(BF16)
        if case["pack"] != "none":
            out["stored"] = _stored(y if case["pack"] == "output" else n)
        return out
    if op == "norm_bwd":
        rstd = s["rstd"][:, None]
        if case["src"] == "act8":
            n = _values(s)
        else:
            n = (s["sum"].float() - (s["mean"][:, None] if s["mean"] is not None else 0.0)) * rstd
        dy = s["dy"].float()
        g = dy * s["gamma"]
        t = g - n * (g * n).mean(1, keepdim=True)
        if case["kind"] == "layer":
            t = t - g.mean(1, keepdim=True)
        dx = t * rstd if s["dx_in"] is None else t * rstd + s["dx_in"].float()
        out = {"dx": dx.to(TYPES[case["dx"]]), "dgamma": (dy * n).sum(0)}
        if case["kind"] == "layer":
            out["dbeta"] = dy.sum(0)
        return out
    if op == "gelu_fwd":
        z = s["z"].float()
        return {"g": (z * _cdf(z)).to(BF16), "stored": _stored(z)}
    if op == "gelu_bwd":
        z = _values(s)
        p = _cdf(z)
        dz = s["dg"].float() * (p + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi)))
        return {"dz": dz.to(BF16), "g": (z * p).to(BF16)}
    if op == "wgrad":
        return {"dw": s["dy"].float().t() @ _values(s)}
    if op == "pack":
        return {"stored": _stored(s["x"].float())}
    v = _values(s)
    return {"y": (v if s["gamma"] is None else v * s["gamma"] + s["beta"]).to(BF16)}


# ------------------------------------------------------------------------------------------------------------ the framework's
def _run_own(s):
    from vita_amd import ops
    case = s["case"]
    op, d = case["op"], s["d"]
    if op == "norm_fwd":
        stream = F32 if s["res"] is not None and F32 in (s["x"].dtype, s["res"].dtype) else BF16
        a = ops.addnorm_fwd(s["x"], s["gamma"], s["beta"], residual=s["res"], kind=case["kind"], eps=s["eps"],
                            y_dtype=BF16 if case["y"] else None, sum_dtype=stream if s["res"] is not None else None,
                            pack=None if case["pack"] == "none" else case["pack"])
        out = {"rstd": a.rstd}
        if a.sum is not None:
            out["sum"] = a.sum[:, :d]
        if a.y is not None:
            out["y"] = a.y[:, :d]
        if a.act is not None:
            out["stored"] = ops.act8_unpack(a.act)[:, :d]
        return out
    if op == "norm_bwd":
        src = ops.Act8(s["q"], s["scale"], d) if case["src"] == "act8" else s["sum"]
        dx, dgamma, dbeta = ops.addnorm_bwd(s["dy"], src, s["rstd"], s["gamma"], kind=case["kind"], mean=s["mean"],
                                            dx_in=s["dx_in"], dx_dtype=TYPES[case["dx"]])
        out = {"dx": dx[:, :d], "dgamma": dgamma}
        if case["kind"] == "layer":
            out["dbeta"] = dbeta
        return out
    if op == "gelu_fwd":
        g, act = ops.gelu_act8_fwd(s["z"])
        return {"g": g[:, :d], "stored": ops.act8_unpack(act)[:, :d]}
    if op == "pack":
        return {"stored": ops.act8_unpack(ops.act8_pack(s["x"]))[:, :d]}
    act = ops.Act8(s["q"], s["scale"], d)
    if op == "gelu_bwd":
        dz, g = ops.gelu_act8_bwd(s["dg"], act)
        return {"dz": dz[:, :d], "g": g[:, :d]}
    if op == "wgrad":
        return {"dw": ops.act8_wgrad(s["dy"], act)}
    return {"y": ops.act8_unpack(act, gamma=s["gamma"], beta=s["beta"])[:, :d]}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------------------------------------ in 64 bits
def _exact_stored(x):
    """Nearest storable number from its spacing: 2^(max(floor(log2 |v|), -6) - 3) for v = x / 2^e."""
    r, d = x.shape
    pad = -d % GROUP
    g = torch.nn.functional.pad(x, (0, pad)).reshape(r, -1, GROUP)
    fine = torch.isfinite(g)
    top = torch.where(fine, g.abs(), torch.zeros_like(g)).amax(-1, keepdim=True)
    e = torch.full_like(top, -117.0)
    for k in range(-117, 120):                      # the smallest of the 237 scales that holds the group
        e = torch.where((top > 448.0 * 2.0 ** k) & (e == k), torch.full_like(e, min(k + 1, 119)), e)
    v = torch.where(fine, g, torch.full_like(g, math.nan)) * torch.exp2(-e)
    v = v.clamp(-448.0, 448.0)
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3.0)
    return (torch.round(v / step) * step * torch.exp2(e)).reshape(r, -1)[:, :d]


def exact(case, seed):
    s = prepare(case, seed)
    op, d = case["op"], case["d"]
    f64 = lambda t: None if t is None else t.double()
    if "q" in s:
        v = s["q"].float().double() * 2.0 ** (s["scale"].view(torch.uint8).double() - 127.0).repeat_interleave(GROUP, 1)
        v = v[:, :d]
    gamma, beta = f64(s.get("gamma")), f64(s.get("beta"))
    if op == "norm_fwd":
        t = f64(s["x"])
        out = {}
        if s["res"] is not None:
            t = out["sum"] = t + f64(s["res"])
        mean = t.sum(1, keepdim=True) / d if case["kind"] == "layer" else 0.0
        var = (t - mean).pow(2).sum(1, keepdim=True) / d
        n = (t - mean) / torch.sqrt(var + s["eps"])
        y = n * gamma + (beta if beta is not None else 0.0)
        out["rstd"] = 1.0 / torch.sqrt(var[:, 0] + s["eps"])
        if case["y"]:
            out["y"] = y
        if case["pack"] != "none":
            out["stored"] = _exact_stored(y if case["pack"] == "output" else n)
        return out
    if op == "norm_bwd":
        rstd, dy = f64(s["rstd"])[:, None], f64(s["dy"])
        n = v if "q" in s else (f64(s["sum"]) - (f64(s["mean"])[:, None] if s["mean"] is not None else 0.0)) * rstd
        g = dy * gamma
        dx = rstd * (g - n * ((g * n).sum(1, keepdim=True) / d))
        out = {"dgamma": torch.sum(dy * n, 0)}
        if case["kind"] == "layer":
            dx = dx - rstd * (g.sum(1, keepdim=True) / d)
            out["dbeta"] = torch.sum(dy, 0)
        out["dx"] = dx if s["dx_in"] is None else dx + f64(s["dx_in"])
        return out
    if op in ("gelu_fwd", "gelu_bwd"):
        z = f64(s["z"]) if op == "gelu_fwd" else v
        tail = 0.5 * torch.erfc(-z / math.sqrt(2.0))
        if op == "gelu_fwd":
            return {"g": z * tail, "stored": _exact_stored(z)}
        return {"dz": f64(s["dg"]) * (tail + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)), "g": z * tail}
    if op == "wgrad":
        return {"dw": torch.matmul(f64(s["dy"]).t(), v)}
    if op == "pack":
        return {"stored": _exact_stored(f64(s["x"]))}
    return {"y": v if gamma is None else v * gamma + beta}
