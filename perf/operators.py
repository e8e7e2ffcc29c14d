"""Cases of the operators around a mixture-of-experts layer's grouped GEMMs, for timing and for comparing.

  norm       RMS norm with the residual's addition; output in 16 bits, or in fp8 with one scale for the
             tensor (what the fp8 grouped GEMMs take) or one for each row
  route      a router's top-k of its logits: experts and weights of each token, rows per expert, the row of
             each (token, slot) pair in the order of the experts, balance loss
  dispatch   copying tokens to the rows of their experts, and its gradient
  combine    the weighted sum of a token's rows, and its gradients
  w4         a grouped GEMM of few rows with 4-bit weights and group scales

Fields: op (above, with "_bwd" for the backward pass), dtype of the activations or logits, and sizes: `rows` or
`tokens`, `h` (hidden size), `experts`, `k` (experts per token; w4: contraction), `n`, `groups`, `group` (weights
per scale). Where `own` is false `run` computes the plain form, in float32 torch operations with one rounding at the
end; where it is true it calls the package.
"""
import importlib
import math
import random

import torch

own = False

DEV = "cuda"
EPS = 1e-6
TYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32, "e4m3": torch.float8_e4m3fn}
TOP = 448.0  # largest e4m3 value
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4, "e4m3": 1}


def _gg():
    return importlib.import_module("groupgemm-cktile-optimized_amd")


def listed():
    return [
        # Serving, decode: the norm before a layer for a handful of sequences. Latency.
        {"name": "norm_decode", "op": "norm", "dtype": "bf16", "rows": 5, "h": 7168, "residual": True, "out": "same"},
        # Prefill or a training forward in fp8: the input of the gate + up projection, all its rows.
        {"name": "norm_fp8", "op": "norm", "dtype": "bf16", "rows": 32768, "h": 7168, "residual": True, "out": "tensor"},
        # Training: gradients of the norm's input and weight, with the residual's gradient added.
        {"name": "norm_bwd", "op": "norm_bwd", "dtype": "bf16", "rows": 16640, "h": 2880, "residual": True},
        # Decode: a router of many experts over one step's tokens. Latency; no loss.
        {"name": "route_decode", "op": "route", "dtype": "fp32", "tokens": 33, "experts": 256, "k": 8, "renormalize": True,
         "balance": False, "padded": False},
        # Training: a batch with padding between its sequences, and the balance loss.
        {"name": "route_train", "op": "route", "dtype": "fp32", "tokens": 32768, "experts": 256, "k": 8, "renormalize": True,
         "balance": True, "padded": True},
        # Training: the gradient of the logits, few experts, 16-bit logits.
        {"name": "route_bwd", "op": "route_bwd", "dtype": "bf16", "tokens": 16640, "experts": 32, "k": 4, "renormalize": True,
         "balance": True, "padded": False},
        # fp8 activations to the rows of their experts: 4096 tokens, 8 experts each.
        {"name": "dispatch_fp8", "op": "dispatch", "dtype": "e4m3", "tokens": 4096, "experts": 32, "k": 8, "h": 7168,
         "padded": False},
        # The layer's output from its experts' rows.
        {"name": "combine", "op": "combine", "dtype": "bf16", "tokens": 4096, "experts": 32, "k": 8, "h": 7168, "padded": False},
        # Training: gradients of the experts' rows and of the router's weights, a padded batch.
        {"name": "combine_bwd", "op": "combine_bwd", "dtype": "bf16", "tokens": 4160, "experts": 32, "k": 4, "h": 2880,
         "padded": True},
        # Decode of one token: eight of the local experts get one row each, the others none.
        {"name": "w4_decode", "op": "w4", "dtype": "bf16", "groups": 32, "rows": 8, "n": 4096, "k": 7168, "group": 128,
         "zeros": False},
        # Decode of a batch: a few rows for each expert, the finest groups, zero points, ragged tiles.
        {"name": "w4_batch", "op": "w4", "dtype": "bf16", "groups": 32, "rows": 250, "n": 2880, "k": 2880, "group": 32,
         "zeros": True},
        # A short prompt: about 60 rows for each of few experts, fp16.
        {"name": "w4_prompt", "op": "w4", "dtype": "fp16", "groups": 8, "rows": 480, "n": 7168, "k": 2048, "group": 64,
         "zeros": False},
    ]


def draw(rng):
    def log_uniform(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    def size(lo, hi, fine):
        s = rng.choice([256, 64, fine])
        return max(s, log_uniform(lo, hi) // s * s)

    while True:
        op = rng.choice(["norm", "norm", "norm_bwd", "route", "route", "route_bwd", "dispatch", "dispatch_bwd", "combine",
                         "combine_bwd", "w4", "w4"])
        c = {"op": op, "dtype": rng.choice(["bf16", "bf16", "fp16"])}
        if op in ("norm", "norm_bwd"):
            c.update(rows=log_uniform(1, 32768), h=size(512, 14336, 8), residual=rng.random() < 0.75)
            if op == "norm":
                c["out"] = rng.choice(["same", "tensor", "row"])
        elif op == "w4":
            groups = log_uniform(1, 64)
            group = rng.choice([32, 64, 128])
            c.update(groups=groups, rows=max(1, int(groups * math.exp(rng.uniform(math.log(0.25), math.log(64))))),
                     n=size(512, 14336, 8), k=size(512, 14336, group) // group * group, group=group, zeros=rng.random() < 0.4)
        else:
            experts = log_uniform(4, 512)
            c.update(tokens=log_uniform(1, 32768), experts=experts, k=min(experts, rng.choice([1, 2, 4, 6, 8])),
                     padded=rng.random() < 0.4)
            if op.startswith("route"):
                c["dtype"] = rng.choice(["fp32", "fp32", "bf16", "fp16"])
                c.update(renormalize=rng.random() < 0.7, balance=rng.random() < 0.7)
            else:
                if op == "dispatch" and rng.random() < 0.4:
                    c["dtype"] = "e4m3"
                c["h"] = size(512, 14336, 16)
        cost = work(c)["bytes"]
        if cost < 1.6e9 and (op != "w4" or c["groups"] * c["n"] * c["k"] < 1.0e9):
            return c


# ---- inputs ----


def _counts(case):
    """Rows of each group of a w4 case: a router's uneven load, the same for every seed but for its order."""
    g, rows = case["groups"], case["rows"]
    rng = random.Random("%d/%d/%d/%d" % (g, rows, case["n"], case["k"]))
    share = [rng.gammavariate(3.0, 1.0) for _ in range(g)]
    cut, at = [0], 0.0
    for s in share[:-1]:
        at += s
        cut.append(int(rows * at / sum(share)))
    cut.append(rows)
    return [b - a for a, b in zip(cut, cut[1:])]


def _randn(gen, *shape):
    return torch.randn(shape, device=DEV, generator=gen)


def _activations(gen, rows, h, dtype):
    """Rows of a residual stream: N(0, 1), some channels several times larger, as trained models have."""
    v = _randn(gen, rows, h)
    v[:, torch.randint(0, h, (max(1, h // 256),), device=DEV, generator=gen)] *= 8.0
    return v.to(TYPE[dtype])


def _logits(gen, tokens, experts, dtype):
    """A router's logits: N(0, 1.5^2) around a bias that makes some experts busier."""
    return (1.5 * _randn(gen, tokens, experts) + 0.5 * _randn(gen, 1, experts)).to(TYPE[dtype])


def _padding(gen, tokens):
    """A batch of sequences of one length, each with padding after its own end: true where a token is real."""
    length = max(1, min(tokens, 512))
    seqs = -(-tokens // length)
    real = torch.randint((length + 1) // 2, length + 1, (seqs, 1), device=DEV, generator=gen)
    return (torch.arange(length, device=DEV)[None, :] < real).reshape(-1)[:tokens].contiguous()


def _pack(q, scales, zeros):
    """The package's storage of 4-bit weights from q [N, K] in 0..15, scales and zeros [N, K / group]: tiles of 16 rows
    by 128 columns, 64 pieces of 16 bytes in each: piece 16 a + r holds row r, its word j the columns 32 j + 8 a .. + 7,
    the even ones in the low half of the word, the odd ones in the high half."""
    n, k = q.shape
    nt, kt = -(-n // 16), -(-k // 128)
    full = torch.zeros(nt * 16, kt * 128, dtype=torch.uint8, device=q.device)
    full[:n, :k] = q
    t = full.view(nt, 16, kt, 4, 4, 4, 2).permute(0, 2, 4, 1, 3, 6, 5).reshape(nt, kt, 64, 16, 2)  # r c j a p o -> a r j o p
    packed = t[..., 0] | (t[..., 1] << 4)

    def tiles(s):
        f = torch.zeros(nt * 16, s.shape[1], dtype=s.dtype, device=s.device)
        f[:n] = s
        return f.view(nt, 16, -1).transpose(1, 2).contiguous()

    return packed, tiles(scales), None if zeros is None else tiles(zeros)


def _w4_weights(gen, case):
    """Weights N(0, 1 / k) of each group in 4 bits: symmetric (zero at 8), or between each group's least and greatest."""
    n, k, group, dtype = case["n"], case["k"], case["group"], TYPE[case["dtype"]]
    packed, scales, zeros = [], [], []
    for _ in range(case["groups"]):
        w = (_randn(gen, n, k) * k**-0.5).view(n, k // group, group)
        if case["zeros"]:
            lo, hi = w.amin(2).clamp(max=0.0), w.amax(2).clamp(min=0.0)
            s = ((hi - lo) / 15).to(dtype)
            z = (-lo / s.float()).round().clamp(0, 15)
        else:
            s = (w.abs().amax(2) / 7.5).to(dtype)
            z = torch.full_like(s, 8, dtype=torch.float32)
        q = (w / s.float()[:, :, None] + z[:, :, None]).round().clamp(0, 15).to(torch.uint8).view(n, k)
        p, s, z = _pack(q, s, z.to(torch.uint8) if case["zeros"] else None)
        packed.append(p)
        scales.append(s)
        zeros.append(z)
    return torch.stack(packed), torch.stack(scales), torch.stack(zeros) if case["zeros"] else None


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    op, dtype = case["op"], case["dtype"]
    s = {"case": case}
    if op.startswith("norm"):
        m, h = case["rows"], case["h"]
        s["weight"] = (1 + 0.2 * _randn(gen, h)).to(TYPE[dtype])
        s["x"] = _activations(gen, m, h, dtype)
        s["residual"] = (4 * _randn(gen, m, h)).to(TYPE[dtype]) if case["residual"] and op == "norm" else None
        if op == "norm_bwd":
            s["rstd"] = (s["x"].float().square().mean(1) + EPS).rsqrt()
            s["grad_y"] = (_randn(gen, m, h) / 64).to(TYPE[dtype])
            s["grad_h"] = (_randn(gen, m, h) / 64).to(TYPE[dtype]) if case["residual"] else None
    elif op == "w4":
        counts = _counts(case)
        random.Random(seed).shuffle(counts)
        s["lens"] = torch.tensor(counts, dtype=torch.int64, device=DEV)
        s["x"] = _randn(gen, case["rows"], case["k"]).to(TYPE[dtype])
        s["packed"], s["scales"], s["zeros"] = _w4_weights(gen, case)
        s["most"], s["active"] = max(counts), sum(c > 0 for c in counts)
    else:
        t, e, k = case["tokens"], case["experts"], case["k"]
        route = op.startswith("route")
        s["logits"] = _logits(gen, t, e, dtype if route else "fp32")
        s["mask"] = _padding(gen, t) if case["padded"] else None
        if op != "route":
            s["routing"] = _plain_route(s["logits"], k, s["mask"], case.get("renormalize", True), case.get("balance", False))
        if op == "route_bwd":
            s["grad_weights"] = _randn(gen, t, k) / 64
            s["grad_loss"] = torch.full((), 0.01, device=DEV) if case["balance"] else None
        elif not route:
            h, pairs = case["h"], op in ("combine", "combine_bwd", "dispatch_bwd")
            v = _activations(gen, t * k if pairs else t, h, "bf16" if dtype == "e4m3" else dtype)
            s["v"] = v.float().clamp(-TOP, TOP).to(TYPE[dtype]) if dtype == "e4m3" else v
            if op == "combine_bwd":
                s["grad_out"] = (_randn(gen, t, h) / 64).to(TYPE[dtype])
    return s


# ---- plain forms ----


def _plain_norm(s):
    case = s["case"]
    h = s["x"] if s["residual"] is None else (s["x"].float() + s["residual"].float()).to(s["x"].dtype)
    v = h.float()
    rstd = (v.square().mean(1) + EPS).rsqrt()
    y = v * rstd[:, None] * s["weight"].float()
    if case["out"] == "same":
        return {"y": y.to(h.dtype), "h": h, "rstd": rstd}
    top = y.abs().amax(1) if case["out"] == "row" else y.abs().amax().reshape(1)
    scale = torch.where(top > 0, top / TOP, torch.ones_like(top))
    q = (y / (scale[:, None] if case["out"] == "row" else scale)).clamp(-TOP, TOP).to(torch.float8_e4m3fn)
    return {"y": q, "h": h, "rstd": rstd, "scale": scale}


def _plain_norm_bwd(s):
    h, g, rstd = s["x"].float(), s["grad_y"].float(), s["rstd"][:, None]
    wg = g * s["weight"].float()
    gx = rstd * wg - h * (rstd.pow(3) * (wg * h).mean(1, keepdim=True))
    if s["grad_h"] is not None:
        gx = gx + s["grad_h"].float()
    return {"grad_x": gx.to(s["x"].dtype), "grad_weight": (g * h * rstd).sum(0).to(s["weight"].dtype)}


def _plain_route(logits, k, mask, renormalize, balance):
    t, e = logits.shape
    v = logits.float()
    live = torch.ones(t, dtype=torch.bool, device=v.device) if mask is None else mask
    top = v.amax(1, keepdim=True)
    ex = (v - top).exp()
    total = ex.sum(1, keepdim=True)
    p = ex / total
    best, order = v.sort(dim=1, descending=True, stable=True)
    best, order = best[:, :k], order[:, :k]
    w = p.gather(1, order)
    if renormalize:
        w = w / w.sum(1, keepdim=True)
    ok = live[:, None].expand(t, k)
    flat = torch.where(ok, order, e).reshape(-1)
    counts = torch.zeros(e + 1, dtype=torch.int64, device=v.device).scatter_add_(0, flat, torch.ones_like(flat))[:e]
    offs = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    place = torch.empty_like(flat)
    place[flat.sort(stable=True).indices] = torch.arange(t * k, device=v.device)
    r = {"experts": torch.where(ok, order, -1).int(), "weights": torch.where(ok, w, 0.0), "counts": counts, "offs": offs,
         "rows": torch.where(ok, place.view(t, k), -1).int(),
         "lse": torch.where(live, (top + total.log())[:, 0], -math.inf)}
    if balance:
        n = live.sum().clamp(min=1).float()
        r["slope"] = counts.float() * e / (counts.sum().clamp(min=1).float() * n)
        r["loss"] = (r["slope"] * (p * live[:, None]).sum(0)).sum()
    return r


def _plain_route_bwd(s):
    r, v = s["routing"], s["logits"].float()
    p = (v - r["lse"][:, None]).exp() if s["mask"] is None else torch.where(s["mask"][:, None], (v - r["lse"][:, None]).exp(), 0.0)
    w, ok = r["weights"], r["experts"] >= 0
    slot = torch.where(ok, r["experts"], 0).long()
    gw = torch.where(ok, s["grad_weights"], 0.0)
    g = torch.zeros_like(v) if s["grad_loss"] is None else (s["grad_loss"] * r["slope"]).expand_as(v)
    if s["case"]["renormalize"]:
        extra = torch.zeros_like(v).scatter_add_(1, slot, w * (gw - (w * gw).sum(1, keepdim=True)))
        out = p * (g - (p * g).sum(1, keepdim=True)) + extra
    else:
        g = torch.scatter_add(g, 1, slot, gw)
        out = p * (g - (p * g).sum(1, keepdim=True))
    return {"grad_logits": out.to(s["logits"].dtype)}


def _plain_rows(s):
    """dispatch, combine and their gradients."""
    op, r, v = s["case"]["op"], s["routing"], s["v"]
    t, k = r["rows"].shape
    ok = r["rows"] >= 0
    at = torch.where(ok, r["rows"], t * k).long()  # one row more than there are: where nothing goes
    token = torch.arange(t, device=v.device)[:, None].expand(t, k)
    if op == "dispatch":
        xs = torch.zeros(t * k + 1, v.shape[1], dtype=v.dtype, device=v.device)
        wide = xs.view(torch.uint8 if v.element_size() == 1 else torch.int16)
        wide[at.reshape(-1)] = v.view(wide.dtype)[token.reshape(-1)]
        return {"xs": xs[:-1]}
    w = r["weights"] if op.startswith("combine") else ok.float()
    if op in ("combine", "dispatch_bwd"):
        part = torch.where(ok, r["rows"], 0).long()
        out = (torch.where(ok[:, :, None], v[part].float(), 0.0) * w[:, :, None]).sum(1)
        return {"out": out.to(v.dtype)}
    g = s["grad_out"].float()
    gy = torch.zeros(t * k + 1, v.shape[1], dtype=v.dtype, device=v.device)
    gy[at.reshape(-1)] = (w[:, :, None] * g[:, None, :]).to(v.dtype).view(t * k, -1)
    part = torch.where(ok, r["rows"], 0).long()
    return {"grad_y": gy[:-1], "grad_weights": torch.where(ok, (v[part].float() * g[:, None, :]).sum(2), 0.0)}


def _unpack(packed, scales, zeros, n, k, group):
    """Float32 weights [.., N, K] of the package's 4-bit storage."""
    a, nt, kt = packed.shape[:3]
    t = packed.view(a, nt, kt, 4, 16, 4, 2, 2)  # a r j o and pairs of p
    q = torch.stack([t & 15, t >> 4], -1)       # .. o, p / 2, p % 2
    q = q.permute(0, 1, 4, 2, 5, 3, 7, 8, 6).reshape(a, nt * 16, kt * 128)[:, :n, :k]

    def rows(s):
        return s.transpose(2, 3).reshape(a, nt * 16, -1)[:, :n, :, None].float()

    w = q.reshape(a, n, k // group, group).float()
    return ((w - (8.0 if zeros is None else rows(zeros))) * rows(scales)).view(a, n, k)


def _plain_w4(s):
    case, lens, x = s["case"], s["lens"], s["x"]
    used = lens > 0
    pick = used.int().sort(descending=True, stable=True).indices[: s["active"]]  # the groups that have rows
    w = _unpack(s["packed"][pick], s["scales"][pick], None if s["zeros"] is None else s["zeros"][pick], case["n"], case["k"],
                case["group"])
    ends = lens.cumsum(0)
    row = torch.arange(x.shape[0], device=x.device)
    g = torch.searchsorted(ends, row, right=True)
    place, rank = (used.cumsum(0) - 1)[g], row - (ends - lens)[g]
    xt = torch.zeros(s["active"], case["k"], s["most"], device=x.device)
    xt[place, :, rank] = x.float()
    return {"out": torch.bmm(w, xt)[place, :, rank].to(x.dtype)}


# ---- calls ----


def _own_routing(gg, s):
    r = s["routing"]
    return gg.Routing(r["experts"], r["weights"], r["counts"], r["offs"], r["rows"], r["lse"], r.get("slope"), r.get("loss"),
                      s["case"].get("renormalize", True))


def _own(s):
    gg, case = _gg(), s["case"]
    op = case["op"]
    if op == "norm":
        quantized = case["out"] != "same"
        y, h, rstd, scale = gg.rms_norm(s["x"], s["weight"], s["residual"], EPS, torch.float8_e4m3fn if quantized else None,
                                        case["out"] if quantized else None)
        return {"y": y, "h": h, "rstd": rstd, "scale": scale} if quantized else {"y": y, "h": h, "rstd": rstd}
    if op == "norm_bwd":
        gx, gw = gg.rms_norm_backward(s["grad_y"], s["x"], s["weight"], s["rstd"], s["grad_h"])
        return {"grad_x": gx, "grad_weight": gw}
    if op == "route":
        r = gg.route(s["logits"], case["k"], s["mask"], case["renormalize"], case["balance"])
        out = {"experts": r.experts, "weights": r.weights, "counts": r.counts, "offs": r.offs, "rows": r.rows, "lse": r.lse}
        return {**out, "slope": r.slope, "loss": r.loss} if case["balance"] else out
    if op == "route_bwd":
        return {"grad_logits": gg.route_backward(s["logits"], _own_routing(gg, s), s["grad_weights"], s["grad_loss"])}
    if op == "dispatch":
        return {"xs": gg.dispatch(s["v"], _own_routing(gg, s))}
    if op == "dispatch_bwd":
        return {"out": gg.dispatch_backward(s["v"], _own_routing(gg, s))}
    if op == "combine":
        return {"out": gg.combine(s["v"], _own_routing(gg, s))}
    if op == "combine_bwd":
        gy, gw = gg.combine_backward(s["grad_out"], s["v"], _own_routing(gg, s))
        return {"grad_y": gy, "grad_weights": gw}
    w4 = gg.W4Weights(s["packed"], s["scales"], s["zeros"], case["n"], case["k"], case["group"])
    return {"out": gg.grouped_gemm_w4(s["x"], w4, s["lens"])}


def run(state):
    if own:
        return _own(state)
    case = state["case"]
    op = case["op"]
    if op == "norm":
        return _plain_norm(state)
    if op == "norm_bwd":
        return _plain_norm_bwd(state)
    if op == "route":
        return _plain_route(state["logits"], case["k"], state["mask"], case["renormalize"], case["balance"])
    if op == "route_bwd":
        return _plain_route_bwd(state)
    if op == "w4":
        return _plain_w4(state)
    return _plain_rows(state)


def work(case):
    op, es = case["op"], SIZE[case["dtype"]]
    if op.startswith("norm"):
        m, h = case["rows"], case["h"]
        if op == "norm_bwd":
            return {"bytes": es * m * h * (4 if case["residual"] else 3) + 4 * m + 2 * es * h, "flops": 12.0 * m * h}
        y = es if case["out"] == "same" else 1
        return {"bytes": m * h * (es * (3 if case["residual"] else 1) + y) + 4 * m + es * h, "flops": 6.0 * m * h}
    if op == "w4":
        n, k, g = case["n"], case["k"], case["group"]
        a = sum(c > 0 for c in _counts(case))
        return {"bytes": a * n * k // 2 + a * n * (k // g) * (3 if case["zeros"] else 2) + es * case["rows"] * (n + k)
                + 8 * case["groups"], "flops": 2.0 * case["rows"] * n * k}
    t, e, k = case["tokens"], case["experts"], case["k"]
    if op == "route":
        return {"bytes": es * t * e + 12 * t * k + 4 * t + 16 * e, "flops": 4.0 * t * e}
    if op == "route_bwd":
        return {"bytes": 2 * es * t * e + 12 * t * k + 4 * t + 4 * e, "flops": 6.0 * t * e}
    h = case["h"]
    moved = es * h * t * (1 + k) + 4 * t * k
    if op == "combine_bwd":
        return {"bytes": moved + es * h * t * k + 8 * t * k, "flops": 3.0 * t * k * h}
    return {"bytes": moved + (4 * t * k if op == "combine" else 0), "flops": 0.0 if op == "dispatch" else 2.0 * t * k * h}


# ---- the same from the definitions, in 64 bits ----


def _exact_route(logits, k, mask, renormalize, balance):
    t, e = logits.shape
    l = logits.double()
    lse = torch.logsumexp(l, 1)
    p = torch.exp(l - lse[:, None])
    live = torch.ones(t, dtype=torch.bool, device=l.device) if mask is None else mask
    chosen = torch.argsort(l, dim=1, descending=True, stable=True)[:, :k]
    w = torch.take_along_dim(p, chosen, 1)
    if renormalize:
        w = w / w.sum(1, keepdim=True)
    w = w * live[:, None]
    hot = torch.zeros(t, e, dtype=torch.float64, device=l.device)
    hot.scatter_(1, chosen, live[:, None].double().expand(t, k).contiguous())
    count = hot.sum(0)
    out = {"experts": None, "weights": w, "counts": None, "offs": None, "rows": None, "lse": torch.where(live, lse, -math.inf)}
    if balance:
        n = max(1, int(live.sum()))
        out["slope"] = e * count / max(1.0, float(count.sum())) / n
        out["loss"] = (out["slope"] @ (p * live[:, None]).sum(0)).reshape(())
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        h = s["x"] if s["residual"] is None else (s["x"].double() + s["residual"].double()).to(s["x"].dtype)
        d = h.double()
        r = 1 / torch.sqrt(torch.mean(d * d, 1) + EPS)
        y = d * r[:, None] * s["weight"].double()
        out = {"h": d, "rstd": r}
        if case["out"] != "same":
            out["scale"] = (y.abs().amax(1) if case["out"] == "row" else y.abs().max().reshape(1)) / TOP
            y = y / (out["scale"][:, None] if case["out"] == "row" else out["scale"])
        out["y"] = y
        return out
    if op == "norm_bwd":
        h, g, w = s["x"].double(), s["grad_y"].double(), s["weight"].double()
        # rstd is an input: the gradient is of h * rstd(h) * w at the rstd given
        r = s["rstd"].double()[:, None]
        inner = torch.sum(g * w * h, 1, keepdim=True) / case["h"]
        gx = r * g * w - h * r**3 * inner
        if s["grad_h"] is not None:
            gx += s["grad_h"].double()
        return {"grad_x": gx, "grad_weight": torch.sum(g * h * r, 0)}
    if op == "route":
        return _exact_route(s["logits"], case["k"], s["mask"], case["renormalize"], case["balance"])
    if op == "route_bwd":
        l, r = s["logits"].double(), s["routing"]
        live = torch.isfinite(r["lse"])
        p = torch.softmax(l, 1) * live[:, None]
        e = torch.clamp(r["experts"], min=0).long()
        gw = s["grad_weights"].double() * (r["experts"] >= 0)
        sel = torch.take_along_dim(p, e, 1)
        gp = torch.zeros_like(l)
        if s["grad_loss"] is not None:
            gp += s["grad_loss"].double() * r["slope"].double()
        if case["renormalize"]:
            total = sel.sum(1, keepdim=True)
            total = torch.where(total > 0, total, 1.0)
            gw = gw / total - (gw * sel).sum(1, keepdim=True) / total**2
        gp.scatter_add_(1, e, gw * (r["experts"] >= 0))
        return {"grad_logits": p * (gp - torch.sum(p * gp, 1, keepdim=True))}
    if op == "w4":
        out, at = torch.empty(case["rows"], case["n"], dtype=torch.float64, device=DEV), 0
        n, k, group = case["n"], case["k"], case["group"]
        row, col = torch.arange(n, device=DEV)[:, None], torch.arange(k, device=DEV)[None, :]
        odd, inside = col % 2, col % 8
        byte = (col // 32 % 4) * 4 + odd * 2 + inside // 4  # of the piece: word, half, byte
        for i, m in enumerate(s["lens"].tolist()):
            if m == 0:
                continue
            piece = s["packed"][i][row // 16, col // 128, (col // 8 % 4) * 16 + row % 16, byte]
            q = torch.where(inside // 2 % 2 == 0, piece & 15, piece >> 4).double()
            z = 8.0 if s["zeros"] is None else s["zeros"][i][row // 16, col // group, row % 16].double()
            w = (q - z) * s["scales"][i][row // 16, col // group, row % 16].double()
            out[at:at + m] = s["x"][at:at + m].double() @ w.T
            at += m
        return {"out": out}
    r, v = s["routing"], s["v"]
    t, k = r["rows"].shape
    if op == "dispatch":
        xs = torch.zeros(t * k, case["h"], dtype=torch.float64, device=DEV)
        for slot in range(k):
            ok = r["rows"][:, slot] >= 0
            xs[r["rows"][ok, slot].long()] = v[ok].double()
        return {"xs": xs}
    if op in ("combine", "dispatch_bwd"):
        out = torch.zeros(t, case["h"], dtype=torch.float64, device=DEV)
        for slot in range(k):
            ok = r["rows"][:, slot] >= 0
            part = v[r["rows"][ok, slot].long()].double()
            out[ok] += part * r["weights"][ok, slot, None].double() if op == "combine" else part
        return {"out": out}
    gy = torch.zeros(t * k, case["h"], dtype=torch.float64, device=DEV)
    gw = torch.zeros(t, k, dtype=torch.float64, device=DEV)
    g = s["grad_out"].double()
    for slot in range(k):
        ok = r["rows"][:, slot] >= 0
        at = r["rows"][ok, slot].long()
        gy[at] = g[ok] * r["weights"][ok, slot, None].double()
        gw[ok, slot] = (g[ok] * v[at].double()).sum(1)
    return {"grad_y": gy, "grad_weights": gw}
