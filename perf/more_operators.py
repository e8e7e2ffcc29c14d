"""Cases of the operators that an expert layer on 8-bit integers needs, for timing and for comparing.

  ln         layer norm with the residual's addition; output in 16 bits, or in int8 with one scale for each row
  ln_bwd     its gradients: of the input, the weight and the bias
  act        the gated activation silu(gate) * up of rows that hold both; output in 16 bits or in int8 rows
  act_bwd    its gradient
  i8         a grouped GEMM in 8-bit integers with a scale for each row of x and each output channel; x in int8 with its
             scales, or in 16 bits, whose rows the call quantizes

Fields: op (above), dtype of the 16-bit side, and sizes: `rows`, `h` (hidden size), `inner` (columns of the activation's
output), `groups`, `n`, `k` (contraction). Where `own` is false `run` computes the plain form, in float32 torch operations
with one rounding at the end; where it is true it calls the package. int8 rows come back as the whole numbers they hold, in
bfloat16 (exact up to 256), beside their scales.
"""
import importlib
import math
import random

import torch

own = False

DEV = "cuda"
EPS = 1e-5
TYPE = {"bf16": torch.bfloat16, "fp16": torch.float16}
TOP = 127.0  # largest value of an int8 row


def _gg():
    return importlib.import_module("groupgemm-cktile-optimized_amd")


def listed():
    return [
        # Serving, decode: the norm before a layer for a handful of sequences. Latency.
        {"name": "ln_decode", "op": "ln", "dtype": "bf16", "rows": 6, "h": 7168, "residual": True, "bias": True, "w32": False,
         "out": "same"},
        # Training forward: the norm of a batch, float32 weights as optimizers keep them.
        {"name": "ln_forward", "op": "ln", "dtype": "bf16", "rows": 32768, "h": 4096, "residual": False, "bias": True,
         "w32": True, "out": "same"},
        # Prefill of an int8 layer: the norm writes the rows and scales that the products read.
        {"name": "ln_i8", "op": "ln", "dtype": "bf16", "rows": 8192, "h": 7168, "residual": True, "bias": True, "w32": False,
         "out": "i8"},
        # Training: gradients of the norm's input, weight and bias, with the residual's gradient added.
        {"name": "ln_bwd", "op": "ln_bwd", "dtype": "bf16", "rows": 16640, "h": 2880, "residual": True, "bias": True,
         "w32": False},
        # Decode: the activation between the two products of a few tokens' experts. Latency.
        {"name": "act_decode", "op": "act", "dtype": "bf16", "rows": 33, "inner": 2048, "out": "i8"},
        # Training forward: the activation of all experts' rows.
        {"name": "act_forward", "op": "act", "dtype": "bf16", "rows": 32768, "inner": 2048, "out": "same"},
        # Prefill of an int8 layer, rows that no power of two divides.
        {"name": "act_i8", "op": "act", "dtype": "fp16", "rows": 16640, "inner": 2880, "out": "i8"},
        # Training: the gradient of gate and up.
        {"name": "act_bwd", "op": "act_bwd", "dtype": "bf16", "rows": 32768, "inner": 2048},
        # Decode of one token: eight of the local experts get one row each, the others none.
        {"name": "i8_decode", "op": "i8", "dtype": "bf16", "groups": 32, "rows": 8, "n": 4096, "k": 7168, "quantized": True},
        # Decode of a batch: a few rows for each expert, ragged, in 16 bits when the call gets them.
        {"name": "i8_batch", "op": "i8", "dtype": "fp16", "groups": 32, "rows": 250, "n": 2880, "k": 2880, "quantized": False},
        # A prompt: about 500 rows for each expert, in 16 bits when the call gets them.
        {"name": "i8_prompt", "op": "i8", "dtype": "bf16", "groups": 8, "rows": 4160, "n": 7168, "k": 2048, "quantized": False},
        # Prefill of a large batch: gate and up of 32768 rows.
        {"name": "i8_prefill", "op": "i8", "dtype": "bf16", "groups": 8, "rows": 32768, "n": 4096, "k": 7168, "quantized": True},
    ]


def draw(rng):
    def log_uniform(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    def size(lo, hi, fine):
        s = rng.choice([256, 64, fine])
        return max(s, log_uniform(lo, hi) // s * s)

    while True:
        op = rng.choice(["ln", "ln", "ln_bwd", "act", "act", "act_bwd", "i8", "i8", "i8"])
        c = {"op": op, "dtype": rng.choice(["bf16", "bf16", "fp16"])}
        if op == "i8":
            groups = log_uniform(1, 64)
            c.update(groups=groups, rows=max(1, int(groups * math.exp(rng.uniform(math.log(0.25), math.log(4096))))),
                     n=size(512, 14336, 8), k=size(512, 14336, 16) // 16 * 16, quantized=rng.random() < 0.6)
            if c["groups"] * c["n"] * c["k"] < 6.0e8 and work(c)["flops"] < 1.9e12:
                return c
            continue
        c["rows"] = log_uniform(1, 32768)
        if op.startswith("ln"):
            c.update(h=size(512, 14336, 8), residual=rng.random() < 0.6, bias=rng.random() < 0.8, w32=rng.random() < 0.4)
        else:
            c["inner"] = size(256, 14336, 8)
        if op in ("ln", "act"):
            c["out"] = rng.choice(["same", "i8"])
        if work(c)["bytes"] < 6.5e8:
            return c


# ---- inputs ----


def _counts(case):
    """Rows of each group: a router's uneven load, the same for every seed but for its order."""
    g, rows = case["groups"], case["rows"]
    rng = random.Random("%d/%d/%d/%d" % (g, rows, case["n"], case["k"]))
    share = [rng.gammavariate(6.0, 1.0) for _ in range(g)]
    cut, at = [0], 0.0
    for s in share[:-1]:
        at += s
        cut.append(int(rows * at / sum(share)))
    cut.append(rows)
    return [b - a for a, b in zip(cut, cut[1:])]


def _randn(gen, *shape):
    return torch.randn(shape, device=DEV, generator=gen)


def _activations(gen, rows, h, dtype):
    """Rows of a residual stream: N(0.1, 1), some channels several times larger, as trained models have."""
    v = _randn(gen, rows, h) + 0.1
    v[:, torch.randint(0, h, (max(1, h // 256),), device=DEV, generator=gen)] *= 8.0
    return v.to(TYPE[dtype])


def _quantized(v):
    """(whole numbers, scales) of the rows of a float32 matrix: scale = max |v| / 127, 1 for a row of zeros."""
    top = v.abs().amax(-1)
    scale = torch.where(top > 0, top / TOP, torch.ones_like(top))
    return (v / scale[..., None]).round().clamp(-TOP, TOP), scale


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    op, dtype = case["op"], case["dtype"]
    s = {"case": case}
    if op.startswith("ln"):
        m, h, wt = case["rows"], case["h"], torch.float32 if case["w32"] else TYPE[dtype]
        s["weight"] = (1 + 0.2 * _randn(gen, h)).to(wt)
        s["bias"] = (0.1 * _randn(gen, h)).to(wt) if case["bias"] else None
        s["x"] = _activations(gen, m, h, dtype)
        s["residual"] = (4 * _randn(gen, m, h)).to(TYPE[dtype]) if case["residual"] and op == "ln" else None
        if op == "ln_bwd":
            s["mean"] = s["x"].float().mean(1)
            s["rstd"] = ((s["x"].float() - s["mean"][:, None]).square().mean(1) + EPS).rsqrt()
            s["grad_y"] = (_randn(gen, m, h) / 64).to(TYPE[dtype])
            s["grad_h"] = (_randn(gen, m, h) / 64).to(TYPE[dtype]) if case["residual"] else None
    elif op.startswith("act"):
        m, n = case["rows"], case["inner"]
        s["gu"] = (1.5 * _randn(gen, m, 2 * n)).to(TYPE[dtype])
        if op == "act_bwd":
            s["grad_y"] = (_randn(gen, m, n) / 64).to(TYPE[dtype])
    else:
        counts = _counts(case)
        random.Random(seed).shuffle(counts)
        s["most"], s["active"] = max(counts), sum(c > 0 for c in counts)
        s["lens"] = torch.tensor(counts, dtype=torch.int64, device=DEV)
        b, m, n, k = case["groups"], case["rows"], case["n"], case["k"]
        x = _activations(gen, m, k, dtype)
        if case["quantized"]:
            q, s["x_scale"] = _quantized(x.float())
            s["x"] = q.to(torch.int8)
        else:
            s["x"] = x
        s["w"] = torch.empty(b, n, k, dtype=torch.int8, device=DEV)
        s["w_scale"] = torch.empty(b, n, device=DEV)
        for i in range(b):  # N(0, 1 / k) weights, a scale for each channel
            q, s["w_scale"][i] = _quantized(_randn(gen, n, k) * k**-0.5)
            s["w"][i] = q.to(torch.int8)
    return s


# ---- plain forms ----


def _plain_ln(s):
    case = s["case"]
    h = s["x"] if s["residual"] is None else (s["x"].float() + s["residual"].float()).to(s["x"].dtype)
    v = h.float()
    mean = v.mean(1)
    v = v - mean[:, None]
    rstd = (v.square().mean(1) + EPS).rsqrt()
    y = v * rstd[:, None] * s["weight"].float()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if case["out"] == "same":
        return {"y": y.to(h.dtype), "h": h, "mean": mean, "rstd": rstd}
    q, scale = _quantized(y)
    return {"y": q.bfloat16(), "h": h, "mean": mean, "rstd": rstd, "scale": scale}


def _plain_ln_bwd(s):
    g, rstd = s["grad_y"].float(), s["rstd"][:, None]
    xh = (s["x"].float() - s["mean"][:, None]) * rstd
    wg = g * s["weight"].float()
    gx = rstd * (wg - wg.mean(1, keepdim=True) - xh * (wg * xh).mean(1, keepdim=True))
    if s["grad_h"] is not None:
        gx = gx + s["grad_h"].float()
    return {"grad_x": gx.to(s["x"].dtype), "grad_weight": (g * xh).sum(0).to(s["weight"].dtype),
            "grad_bias": g.sum(0).to(s["weight"].dtype)}


def _plain_act(s):
    gate, up = s["gu"].float().chunk(2, dim=1)
    y = gate * torch.sigmoid(gate) * up
    if s["case"]["out"] == "same":
        return {"y": y.to(s["gu"].dtype)}
    q, scale = _quantized(y)
    return {"y": q.bfloat16(), "scale": scale}


def _plain_act_bwd(s):
    gate, up = s["gu"].float().chunk(2, dim=1)
    p, g = torch.sigmoid(gate), s["grad_y"].float()
    return {"grad_gu": torch.cat([g * up * p * (1 + gate * (1 - p)), g * gate * p], dim=1).to(s["gu"].dtype)}


def _plain_i8(s):
    case, lens = s["case"], s["lens"]
    q, scale = (s["x"].float(), s["x_scale"]) if case["quantized"] else _quantized(s["x"].float())
    used = lens > 0
    pick = used.int().sort(descending=True, stable=True).indices[: s["active"]]  # the groups that have rows
    w = s["w"][pick].float() * s["w_scale"][pick][:, :, None]
    ends = lens.cumsum(0)
    row = torch.arange(q.shape[0], device=q.device)
    g = torch.searchsorted(ends, row, right=True)
    place, rank = (used.cumsum(0) - 1)[g], row - (ends - lens)[g]
    xt = torch.zeros(s["active"], case["k"], s["most"], device=q.device)
    xt[place, :, rank] = q
    out = torch.bmm(w, xt)[place, :, rank] * scale[:, None]
    return {"out": out.to(TYPE[case["dtype"]])}


# ---- calls ----


def _own(s):
    gg, case = _gg(), s["case"]
    op = case["op"]
    if op == "ln":
        i8 = case["out"] == "i8"
        y, h, mean, rstd, scale = gg.layer_norm(s["x"], s["weight"], s["bias"], s["residual"], EPS,
                                                torch.int8 if i8 else None, "row" if i8 else None)
        out = {"y": y.bfloat16() if i8 else y, "h": h, "mean": mean, "rstd": rstd}
        return {**out, "scale": scale} if i8 else out
    if op == "ln_bwd":
        gx, gw, gb = gg.layer_norm_backward(s["grad_y"], s["x"], s["weight"], s["mean"], s["rstd"], s["grad_h"])
        return {"grad_x": gx, "grad_weight": gw, "grad_bias": gb}
    if op == "act":
        if case["out"] == "same":
            return {"y": gg.silu_product(s["gu"]).y}
        y, scale = gg.silu_product(s["gu"], torch.int8)
        return {"y": y.bfloat16(), "scale": scale}
    if op == "act_bwd":
        return {"grad_gu": gg.silu_product_backward(s["grad_y"], s["gu"])}
    w = gg.I8Weights(s["w"], s["w_scale"])
    if case["quantized"]:
        return {"out": gg.grouped_gemm_i8(s["x"], w, s["lens"], s["x_scale"], TYPE[case["dtype"]])}
    return {"out": gg.grouped_gemm_i8(s["x"], w, s["lens"])}


def run(state):
    if own:
        return _own(state)
    return {"ln": _plain_ln, "ln_bwd": _plain_ln_bwd, "act": _plain_act, "act_bwd": _plain_act_bwd,
            "i8": _plain_i8}[state["case"]["op"]](state)


def work(case):
    op, m = case["op"], case["rows"]
    if op.startswith("ln"):
        h, ws = case["h"], 4 if case["w32"] else 2
        if op == "ln_bwd":
            return {"bytes": 2 * m * h * (4 if case["residual"] else 3) + 8 * m + 3 * ws * h, "flops": 14.0 * m * h}
        y = 2 if case["out"] == "same" else 1
        return {"bytes": m * h * ((6 if case["residual"] else 2) + y) + (8 if y == 2 else 12) * m + ws * h * (2 if case["bias"] else 1),
                "flops": 8.0 * m * h}
    if op == "act":
        return {"bytes": m * case["inner"] * (6 if case["out"] == "same" else 5) + (0 if case["out"] == "same" else 4 * m),
                "flops": 6.0 * m * case["inner"]}
    if op == "act_bwd":
        return {"bytes": 10 * m * case["inner"], "flops": 12.0 * m * case["inner"]}
    n, k = case["n"], case["k"]
    a = sum(c > 0 for c in _counts(case))
    return {"bytes": a * n * (k + 4) + m * (k + 4 if case["quantized"] else 2 * k) + 2 * m * n + 8 * case["groups"],
            "flops": 2.0 * m * n * k}


# ---- the same from the definitions, in 64 bits ----


def _exact_rows(v):
    """Whole numbers and scales of float64 rows."""
    top = torch.amax(torch.abs(v), 1)
    scale = torch.where(top == 0, 1.0, top / TOP)
    return torch.round(v / scale[:, None]), scale


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op.startswith("ln"):
        w = s["weight"].double()
        if op == "ln_bwd":
            # mean and rstd are inputs: the gradient is of (h - mean) * rstd * w at the values given
            d = s["x"].double() - s["mean"].double()[:, None]
            r, g = s["rstd"].double()[:, None], s["grad_y"].double()
            inner = torch.sum(g * w * d, 1, keepdim=True) / case["h"]
            gx = r * (g * w - torch.sum(g * w, 1, keepdim=True) / case["h"]) - d * r**3 * inner
            if s["grad_h"] is not None:
                gx += s["grad_h"].double()
            return {"grad_x": gx, "grad_weight": torch.sum(g * d * r, 0), "grad_bias": torch.sum(g, 0)}
        h = s["x"] if s["residual"] is None else (s["x"].double() + s["residual"].double()).to(s["x"].dtype)
        d = h.double()
        var, mean = torch.var_mean(d, 1, correction=0)
        r = 1 / torch.sqrt(var + EPS)
        y = (d - mean[:, None]) * r[:, None] * w
        if s["bias"] is not None:
            y += s["bias"].double()
        out = {"y": y, "h": d, "mean": mean, "rstd": r}
        if case["out"] == "i8":
            out["y"], out["scale"] = _exact_rows(y)
        return out
    if op.startswith("act"):
        n = case["inner"]
        a, b = s["gu"][:, :n].double(), s["gu"][:, n:].double()
        e = torch.exp(-a)
        if op == "act":
            y = a * b / (1 + e)
            if case["out"] == "same":
                return {"y": y}
            q, scale = _exact_rows(y)
            return {"y": q, "scale": scale}
        g = s["grad_y"].double()
        return {"grad_gu": torch.hstack([g * b * (1 + e + a * e) / (1 + e) ** 2, g * a / (1 + e)])}
    out, at = torch.empty(case["rows"], case["n"], dtype=torch.float64, device=DEV), 0
    q, scale = (s["x"].double(), s["x_scale"].double()) if case["quantized"] else _exact_rows(s["x"].double())
    for i, m in enumerate(s["lens"].tolist()):
        if m == 0:
            continue
        out[at:at + m] = (q[at:at + m] @ s["w"][i].double().T) * scale[at:at + m, None] * s["w_scale"][i].double()
        at += m
    return {"out": out}
