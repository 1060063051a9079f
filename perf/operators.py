"""What the framework's row-wise and training operators are timed on: root-mean-square norm (with the residual's addition, with an
8-bit output), the gated projection (training, serving, 8-bit operands) and gradient clipping by the global norm.

`run` computes a case in plain torch operations, or through the framework's own operators where `own` is true."""
import math
import os
import sys

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}
_E4M3_MAX = 448.0
_EPS = 1e-6

# the gradient tensors of the 256-pixel student that the framework trains (110 tensors, 5.6 M values): element counts
_STUDENT = ([262144, 512] * 8 + [2464, 213444, 78848, 154, 1, 154, 3, 462, 78848, 154] + [213444, 78848, 154, 1, 154] * 8
            + [106722, 78848, 154, 1, 77, 53361, 39424, 77, 1, 77, 27027, 39424, 77, 1, 39, 13689, 19968, 39, 1, 39]
            + [3, 462, 78848, 154] * 4 + [3, 231, 39424, 77, 3, 117, 19968, 39])


def listed():
    return [
        # the mapping network's latent rows at the benchmark's batch: one launch each way, so latency counts
        {"name": "norm_train_latent", "op": "norm_train", "rows": 16, "dim": 512, "dtype": "f32", "weight": "f32", "residual": True, "extra": 0},
        # a long sequence of wide rows, trained in bf16 with fp32 norm weights
        {"name": "norm_train_long", "op": "norm_train", "rows": 16384, "dim": 4096, "dtype": "bf16", "weight": "f32", "residual": True, "extra": 0},
        # one decoded token, quantised for an 8-bit product
        {"name": "norm_quant_token", "op": "norm_quant", "rows": 1, "dim": 2048, "dtype": "bf16", "weight": "bf16", "residual": True, "extra": 0},
        # a ragged prefill, rows of a wider buffer
        {"name": "norm_quant_prefill", "op": "norm_quant", "rows": 8191, "dim": 5120, "dtype": "bf16", "weight": "bf16", "residual": True, "extra": 64},
        # the rows that the mean latent is taken over, in the framework's own fp32
        {"name": "gated_train_f32", "op": "gated_train", "rows": 4096, "k": 512, "n": 2048, "dtype": "f32", "act": "gelu", "bias": True, "extra": 0},
        # a feed-forward block of ordinary width on many tokens: bound by the matrix cores
        {"name": "gated_train_bf16", "op": "gated_train", "rows": 8192, "k": 2048, "n": 8192, "dtype": "bf16", "act": "silu", "bias": False, "extra": 0},
        # the same block decoding one token: bound by the weights' bytes
        {"name": "gated_token", "op": "gated", "rows": 1, "k": 4096, "n": 8192, "dtype": "bf16", "act": "silu", "bias": False, "extra": 0},
        # a ragged batch with sizes that no tile divides and rows of no alignment
        {"name": "gated_odd", "op": "gated", "rows": 77, "k": 1001, "n": 2731, "dtype": "f16", "act": "gelu", "bias": True, "extra": 0},
        # a batch of sequences decoding in 8 bits
        {"name": "gated_e4m3_decode", "op": "gated_e4m3", "rows": 16, "k": 4096, "n": 8192, "act": "silu", "bias": False},
        # a prefill in 8 bits
        {"name": "gated_e4m3_prefill", "op": "gated_e4m3", "rows": 8000, "k": 4096, "n": 8192, "act": "silu", "bias": False},
        # the framework's own student: many small tensors
        {"name": "clip_student", "op": "clip", "tensors": 0, "numel": sum(_STUDENT), "dtype": "f32", "norm": "2"},
        # the gradients of a model of half a billion parameters
        {"name": "clip_large", "op": "clip", "tensors": 200, "numel": 500_000_000, "dtype": "bf16", "norm": "2"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """mostly a multiple of 64, as widths are; one in four of any value, odd ones among them"""
    n = _log(rng, lo, hi)
    return n if rng.random() < 0.25 else max(64, n // 64 * 64)


def draw(rng):
    op = rng.choice(["norm_train", "norm_quant", "gated_train", "gated", "gated_e4m3", "clip"])
    dtype = rng.choice(["f32", "f16", "bf16", "bf16"])
    act = rng.choice(["silu", "gelu"])
    if op in ("norm_train", "norm_quant"):
        dim = _width(rng, 64, 8192)
        rows = _log(rng, 1, min(16384, (30 << 20) // dim))
        return {"op": op, "rows": rows, "dim": dim, "dtype": dtype, "weight": rng.choice(["f32", dtype]), "residual": rng.random() < 0.7,
                "extra": rng.choice([0, 0, 64, 3])}
    if op == "gated_train":
        k, n = _width(rng, 64, 4096), _width(rng, 64, 8192)
        most = (8192 * 2048 * 8192) // (16 if dtype == "f32" else 1)
        return {"op": op, "rows": _log(rng, 1, min(8192, max(1, most // (k * n)))), "k": k, "n": n, "dtype": dtype, "act": act,
                "bias": rng.random() < 0.5, "extra": rng.choice([0, 0, 64, 3])}
    if op == "gated":
        return {"op": op, "rows": _log(rng, 1, 512), "k": _width(rng, 64, 4096), "n": _width(rng, 64, 8192), "dtype": dtype, "act": act,
                "bias": rng.random() < 0.5, "extra": rng.choice([0, 0, 64, 3])}
    if op == "gated_e4m3":
        return {"op": op, "rows": _log(rng, 1, 8000), "k": _width(rng, 64, 4096), "n": _width(rng, 64, 8192), "act": act, "bias": rng.random() < 0.5}
    return {"op": "clip", "tensors": _log(rng, 1, 400), "numel": _log(rng, 4000, 250_000_000), "dtype": dtype, "norm": rng.choice(["2", "2", "inf"])}


# ---- inputs ---------------------------------------------------------------------------------------------------------------------
def _rows(g, rows, width, extra, dtype, scale=1.0):
    """[rows, width] of normal values; `extra`: a view into a buffer whose rows are that much longer"""
    t = torch.randn(rows, width + extra, device="cuda", generator=g, dtype=torch.float32)
    return (t * scale).to(dtype)[:, :width]


def _e4m3_rows(t):
    scale = t.abs().amax(-1) / _E4M3_MAX
    return (t / scale[:, None]).to(torch.float8_e4m3fn), scale


def _sizes(case):
    """element counts of a clip case's tensors: the student's, or from tiny biases to large matrices, adding up to `numel`"""
    if case["tensors"] == 0:
        return list(_STUDENT)
    w = [1.0 if i % 3 == 0 else (0.0005 if i % 3 == 1 else 0.31) for i in range(case["tensors"])]
    s = [max(1, int(case["numel"] * x / sum(w))) for x in w]
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, s = case["op"], dict(case)
    if op in ("norm_train", "norm_quant"):
        dt, wdt = _DTYPES[case["dtype"]], _DTYPES[case["weight"]]
        rows, dim = case["rows"], case["dim"]
        s["x"] = _rows(g, rows, dim, case["extra"], dt, 2.0)
        s["r"] = _rows(g, rows, dim, 0, dt, 4.0) if case["residual"] else None
        s["w"] = (1.0 + 0.2 * torch.randn(dim, device="cuda", generator=g)).to(wdt)
        if op == "norm_train":
            s["dy"] = _rows(g, rows, dim, 0, dt, 0.1)
            s["dh"] = _rows(g, rows, dim, 0, dt, 0.1) if case["residual"] else None
            for k in ("x", "r", "w"):
                if s[k] is not None:
                    s[k].requires_grad_(True)
    elif op in ("gated_train", "gated"):
        dt = _DTYPES[case["dtype"]]
        rows, k, n = case["rows"], case["k"], case["n"]
        s["x"] = _rows(g, rows, k, case["extra"], dt)
        s["w"] = _rows(g, 2 * n, k, 0, dt)                       # unit-variance weights, scaled at run time: the equalised learning rate
        s["b"] = (0.1 * torch.randn(2 * n, device="cuda", generator=g)).to(dt) if case["bias"] else None
        s["scale"] = 1 / math.sqrt(k)
        if op == "gated_train":
            s["dy"] = _rows(g, rows, n, 0, dt, 0.1)
            for key in ("x", "w", "b"):
                if s[key] is not None:
                    s[key].requires_grad_(True)
    elif op == "gated_e4m3":
        rows, k, n = case["rows"], case["k"], case["n"]
        s["x"], s["sx"] = _e4m3_rows(_rows(g, rows, k, 0, torch.float32))
        s["w"], s["sw"] = _e4m3_rows(_rows(g, 2 * n, k, 0, torch.float32, 1 / math.sqrt(k)))
        s["b"] = (0.1 * torch.randn(2 * n, device="cuda", generator=g)).to(torch.bfloat16) if case["bias"] else None
    else:
        dt, sizes = _DTYPES[case["dtype"]], _sizes(case)
        off, at = [], 0
        for n in sizes:                                          # one flat buffer, every tensor at a 16-byte boundary: how the graphed step keeps them
            off.append(at)
            at += (n + 7) // 8 * 8
        s["flat"] = torch.zeros(at, device="cuda", dtype=dt)
        s["grads"] = [s["flat"][o:o + n] for o, n in zip(off, sizes)]
        noise = torch.randn(at, device="cuda", dtype=dt, generator=g) * 0.01
        for i, t in enumerate(s["grads"]):
            t.copy_(noise[off[i]:off[i] + sizes[i]] if i % 5 else noise[off[i]:off[i] + sizes[i]] * 8)
        s["params"] = []
        for t in s["grads"]:
            p = torch.nn.Parameter(torch.empty_like(t))
            p.grad = t
            s["params"].append(p)
        # a threshold that the gradients exceed, lowered a little with every pass: a pass then always clips, where a second call
        # with the same threshold would find its gradients clipped already
        s["max_norm"] = [0.5 * 0.01 * (math.sqrt(sum(sizes)) if case["norm"] == "2" else 1.0)]
    return s


# ---- the operators --------------------------------------------------------------------------------------------------------------
def _op():
    if "cagc" not in sys.modules:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "content-aware-gan-compression_amd"))
    import cagc.op
    return cagc.op


def _act(name, g):
    """(act(g), act'(g))"""
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    c = 0.5 * (1 + torch.erf(g * (0.5 ** 0.5)))
    return g * c, c + g * torch.exp(-0.5 * g * g) * (1 / math.sqrt(2 * math.pi))


def _norm_forward(x, r, w, wide):
    """(h as it is returned, h in the wide type, 1 / rms, y in the wide type); the norm reads h as it is returned"""
    h = x if r is None else (x.to(wide) + r.to(wide)).to(x.dtype)
    hf = h.to(wide)
    inv = torch.rsqrt(hf.square().mean(-1, keepdim=True) + _EPS)
    return h, hf, inv, hf * inv * w.to(wide)


def _norm_train(s, wide):
    with torch.no_grad():
        x, r, w = s["x"].detach(), s["r"], s["w"].detach()
        h, hf, inv, y = _norm_forward(x, r, w, wide)
        dy = s["dy"].to(wide)
        gw = dy * w.to(wide)
        xhat = hf * inv
        dx = inv * (gw - xhat * (gw * xhat).mean(-1, keepdim=True))
        dw = (dy * xhat).sum(0)
        if r is None:
            return {"y": y, "dx": dx, "dw": dw}
        dx = dx + s["dh"].to(wide)
        return {"y": y, "h": h, "dx": dx, "dr": dx, "dw": dw}


def _norm_quant(s, wide):
    h, _, _, y = _norm_forward(s["x"], s["r"], s["w"], wide)
    scale = y.abs().amax(-1).div(_E4M3_MAX).clamp_min(2.0 ** -126)
    q = y / scale[..., None]
    return {"q": q, "scale": scale} if s["r"] is None else {"q": q, "scale": scale, "h": h}


def _gated(s, wide):
    z = s["x"].detach().to(wide) @ s["w"].detach().to(wide).t()
    if s["op"] == "gated_e4m3":
        z = z * s["sx"].to(wide)[:, None] * s["sw"].to(wide)[None, :]
    else:
        z = z * s["scale"]
    if s["b"] is not None:
        z = z + s["b"].detach().to(wide)
    g, u = z.chunk(2, -1)
    a, da = _act(s["act"], g)
    return a * u, a, da, u


def _gated_train(s, wide):
    with torch.no_grad():
        y, a, da, u = _gated(s, wide)
        dy = s["dy"].to(wide)
        dz = torch.cat([dy * u * da, dy * a], -1)
        out = {"y": y, "dx": (dz @ s["w"].detach().to(wide)) * s["scale"], "dw": (dz.t() @ s["x"].detach().to(wide)) * s["scale"]}
        if s["b"] is not None:
            out["db"] = dz.sum(0)
        return out


def _total_norm(grads, kind):
    if kind == "inf":
        return torch.stack([t.abs().amax().double() for t in grads]).amax()
    return torch.stack([t.double().square().sum() for t in grads]).sum().sqrt()


def _as(values, types):
    return {k: v if types.get(k) is None else v.to(types[k]) for k, v in values.items()}


def _types(s):
    """the types in which an operator returns its outputs"""
    op = s["op"]
    if op == "norm_train":
        return {"y": s["x"].dtype, "h": s["x"].dtype, "dx": s["x"].dtype, "dr": s["x"].dtype, "dw": s["w"].dtype}
    if op == "norm_quant":
        return {"q": torch.float8_e4m3fn, "scale": torch.float32, "h": s["x"].dtype}
    return {k: s["x"].dtype for k in ("y", "dx", "dw", "db")}


def _run_own(s):
    op, F = s["op"], _op()
    if op == "norm_train":
        if s["r"] is None:
            y = F.rms_norm(s["x"], s["w"], eps=_EPS)
            dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])
            return {"y": y, "dx": dx, "dw": dw}
        y, h = F.rms_norm(s["x"], s["w"], residual=s["r"], eps=_EPS)
        dx, dr, dw = torch.autograd.grad((y, h), (s["x"], s["r"], s["w"]), (s["dy"], s["dh"]))
        return {"y": y, "h": h, "dx": dx, "dr": dr, "dw": dw}
    if op == "norm_quant":
        out = F.rms_norm_e4m3(s["x"], s["w"], residual=s["r"], eps=_EPS)
        return dict(zip(("q", "scale", "h"), out))
    if op == "gated_train":
        y = F.gated_linear(s["x"], s["w"], s["b"], activation=s["act"], scale=s["scale"])
        keys = ("x", "w") if s["b"] is None else ("x", "w", "b")
        grads = torch.autograd.grad(y, [s[k] for k in keys], s["dy"])
        return {"y": y, **{"d" + k: v for k, v in zip(keys, grads)}}
    if op == "gated":
        return {"y": F.gated_linear(s["x"], s["w"], s["b"], activation=s["act"], scale=s["scale"])}
    if op == "gated_e4m3":
        return {"y": F.gated_linear_e4m3(s["x"], s["sx"], s["w"], s["sw"], s["b"], activation=s["act"])}
    s["max_norm"][0] *= 0.9999
    norm = F.clip_grad_norm_(s["params"], s["max_norm"][0], norm_type=float(s["norm"]))
    return {"norm": norm, "grads": s["flat"]}


def run(state):
    s, op = state, state["op"]
    if own:
        return _run_own(s)
    if op == "norm_train":
        return _as(_norm_train(s, torch.float32), _types(s))
    if op == "norm_quant":
        return _as(_norm_quant(s, torch.float32), _types(s))
    if op == "gated_train":
        return _as(_gated_train(s, torch.float32), _types(s))
    if op in ("gated", "gated_e4m3"):
        y = _gated(s, torch.float32)[0]
        return {"y": y.to(torch.bfloat16 if op == "gated_e4m3" else s["x"].dtype)}
    s["max_norm"][0] *= 0.9999
    norm = _total_norm(s["grads"], s["norm"])
    coef = (s["max_norm"][0] / (norm + 1e-6)).clamp(max=1.0)
    for t in s["grads"]:
        t.copy_(t.float() * coef.float())
    return {"norm": norm.float(), "grads": s["flat"]}


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------------
def work(case):
    op = case["op"]
    if op in ("norm_train", "norm_quant"):
        n, e = case["rows"] * case["dim"], _SIZE[case["dtype"]]
        w = case["dim"] * _SIZE[case["weight"]]
        res = 1 if case["residual"] else 0
        if op == "norm_train":      # reads x, dy (and r, dh), writes y, dx (and h); the weight and its gradient
            return {"bytes": n * e * (4 + 3 * res) + 2 * w, "flops": 14 * n}
        return {"bytes": n * e * (1 + 2 * res) + n + 4 * case["rows"] + w, "flops": 7 * n}
    if op in ("gated_train", "gated", "gated_e4m3"):
        m, k, n = case["rows"], case["k"], case["n"]
        e = 1 if op == "gated_e4m3" else _SIZE[case["dtype"]]
        b = 2 * n * (2 if op == "gated_e4m3" else e) if case["bias"] else 0
        if op == "gated_train":     # forward, then the products for dx and dw from saved pre-activations
            return {"bytes": 2 * e * (m * k + 2 * n * k + m * n) + 2 * b, "flops": 12 * m * n * k}
        extra = 4 * (m + 2 * n) if op == "gated_e4m3" else 0
        return {"bytes": e * (m * k + 2 * n * k) + m * n * (2 if op == "gated_e4m3" else e) + b + extra, "flops": 4 * m * n * k}
    n = sum(_sizes(case))
    return {"bytes": 2 * n * _SIZE[case["dtype"]], "flops": 3 * n}


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------------------
def exact(case, seed):
    s, wide = prepare(case, seed), torch.float64
    op = case["op"]
    with torch.no_grad():
        if op in ("norm_train", "norm_quant"):
            x, w = s["x"].to(wide), s["w"].to(wide)
            h = x if s["r"] is None else x + s["r"].to(wide)
            read = h.to(s["x"].dtype).to(wide)               # the sum as it is handed on, which is what is normed
            d = read.shape[-1]
            rms = ((read * read).sum(-1, keepdim=True) / d + _EPS) ** 0.5
            y = read / rms * w
            if op == "norm_quant":
                top = y.abs().max(-1).values / _E4M3_MAX
                out = {"q": y / top[:, None], "scale": top}
                return out if s["r"] is None else {**out, "h": h}
            dy = s["dy"].to(wide)
            t = dy * w
            dx = t / rms - read * ((t * read).sum(-1, keepdim=True) / (d * rms ** 3))
            dw = ((dy * read) / rms).sum(0)
            if s["r"] is None:
                return {"y": y, "dx": dx, "dw": dw}
            dx = dx + s["dh"].to(wide)
            return {"y": y, "h": h, "dx": dx, "dr": dx, "dw": dw}
        if op in ("gated_train", "gated", "gated_e4m3"):
            x, w = s["x"].to(wide), s["w"].to(wide)
            if op == "gated_e4m3":
                x, w = x * s["sx"].to(wide)[:, None], w * s["sw"].to(wide)[:, None]
            else:
                w = w * s["scale"]
            n = case["n"]
            g, u = torch.matmul(x, w[:n].t().contiguous()), torch.matmul(x, w[n:].t().contiguous())
            if s["b"] is not None:
                g, u = g + s["b"][:n].to(wide), u + s["b"][n:].to(wide)
            if case["act"] == "silu":
                e = 1 / (1 + torch.exp(-g))
                a, da = g * e, e + g * e * (1 - e)
            else:
                e = torch.special.ndtr(g)
                a, da = g * e, e + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
            if op != "gated_train":
                return {"y": a * u}
            dy = s["dy"].to(wide)
            dg, du = dy * u * da, dy * a
            out = {"y": a * u, "dx": dg @ w[:n] + du @ w[n:]}
            dgt, dut = dg.t().contiguous(), du.t().contiguous()
            out["dw"] = torch.cat([dgt @ x, dut @ x]) * s["scale"]
            if s["b"] is not None:
                out["db"] = torch.cat([dg.sum(0), du.sum(0)])
            return out
        flat = s["flat"]
        if case["norm"] == "inf":
            norm = flat.abs().max().to(wide)
        else:
            norm = sum(c.to(wide).square().sum() for c in flat.split(1 << 26)) ** 0.5
        threshold = s["max_norm"][0] * 0.9999
        return {"norm": norm, "grads": flat.to(wide) * min(1.0, threshold / (float(norm) + 1e-6))}
