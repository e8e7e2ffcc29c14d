"""The operators around the grouped GEMM in a mixture-of-experts layer, for torch tensors, over the C
ABI in include/gg_moe_layer.h: RMS norm with the residual's addition and an fp8 output, router with
balance loss, dispatch and combine of the experts' rows, grouped products with 4-bit weights.

Every function enqueues its kernels on the current stream of its tensors' device, or on `stream` (a
raw hipStream_t handle), and returns without waiting (but grouped_gemm_w4 with host group sizes, which
copies them to the device and waits for that). Outputs and workspaces come from torch's allocator, from
the memory of the stream that the kernels run on. With `stream`, the caller orders that stream after
whatever wrote the inputs, and what reads the outputs on another stream after it; the allocator is told
of both streams' uses, so a tensor may be dropped before the work is done.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import GG_OK, DType, GGError, _device_sizes, load_library

_T16 = {torch.bfloat16: int(DType.BF16), torch.float16: int(DType.FP16)}
_T8 = {torch.float8_e4m3fn: int(DType.FP8_E4M3), torch.float8_e5m2: int(DType.FP8_E5M2)}
_FP32 = 4  # GG_DTYPE_FP32
_NORM_WORKSPACE = 8192  # GG_NORM_WORKSPACE
_PLAIN, _TENSOR, _ROW, _GIVEN = 0, 1, 2, 3  # gg_norm_scale


_lib = load_library()
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice


def _call(fn, dev, args) -> None:
    """fn(*args, stream) on the current stream of `dev`, with `dev` the current device."""
    current = _raw_stream(dev.index)
    if dev.index == _current_device():
        st = fn(*args, current)
    else:
        with torch.cuda.device(dev):
            st = fn(*args, current)
    if st != GG_OK:
        raise GGError(st, _lib.gg_layer_last_error().decode())


def _tensors(values):
    for v in values:
        if isinstance(v, torch.Tensor):
            yield v
        elif isinstance(v, tuple):
            yield from _tensors(v)


def _on(stream: int, f, *args):
    """f(*args) with `stream` as torch's current one. Memory that torch hands out belongs to its current stream: a
    dropped tensor's block is given out again while work queued there still uses it. So outputs and workspaces of
    kernels on `stream` have to be allocated with that stream current, or nothing would order them after that work."""
    dev = args[0].device
    if dev.type != "cuda":
        return f(*args)  # refused there
    current = torch.cuda.current_stream(dev)
    if stream == current.cuda_stream:
        return f(*args)
    # (handle 0 is the default stream)
    other = torch.cuda.ExternalStream(stream, device=dev) if stream else torch.cuda.default_stream(dev)
    with torch.cuda.stream(other):
        out = f(*args)
    for t in _tensors(args):
        if t.is_cuda:
            t.record_stream(other)
    for t in _tensors((out,)):
        t.record_stream(current)  # what the caller reads there
    return out


def _matrix(name: str, t):
    """Row stride of a device matrix whose rows are contiguous."""
    if t.dim() != 2 or not t.is_cuda:
        raise ValueError(f"{name} must be a device matrix")
    rows, cols = t.stride()
    if cols != 1 and t.shape[1] > 1:
        raise ValueError(f"{name} must have contiguous rows")
    return rows


def _flat(name: str, t, dtype, shape, dev) -> None:
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}")
    if t.shape != shape or t.device != dev or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous tensor of shape {list(shape)} on {dev}")


def _like(name: str, t, ref) -> None:
    if t.dtype != ref.dtype or t.shape != ref.shape or t.device != ref.device:
        raise ValueError(f"{name} must have the type, shape and device of its counterpart")


def _out(t, dtype, shape, dev):
    if t is None:
        return torch.empty(shape, dtype=dtype, device=dev)
    _flat("out", t, dtype, shape, dev)
    return t


def _new_like(x):
    """A contiguous tensor of x's type and shape (empty_like is the quicker of the two)."""
    return torch.empty_like(x) if x.is_contiguous() else torch.empty(x.shape, dtype=x.dtype, device=x.device)


def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


# ---- RMS norm ----


class NormOutput(NamedTuple):
    """rms_norm's outputs: y; h = x + residual (x itself without one); rstd [M] float32; scale float32
    ([1], or [M] for one a row) of an fp8 y, which stands for y * scale, else None."""
    y: "torch.Tensor"
    h: "torch.Tensor"
    rstd: "torch.Tensor"
    scale: "Optional[torch.Tensor]"


def rms_norm(x, weight, residual=None, eps: float = 1e-6, out_dtype=None, scale=None, out=None, out_h=None,
             stream: Optional[int] = None) -> NormOutput:
    """y = h * rsqrt(mean(h^2) + eps) * weight over the rows of h = x + residual (gg_rms_norm).

    x, residual: [M, H] bf16 or fp16, rows contiguous at any stride; weight [H] of x's type or float32.
    out_dtype float8_e4m3fn or float8_e5m2 gives an fp8 y: with one scale for the tensor (scale=None or
    "tensor": the x_scale of grouped_gemm_fp8), one for each row ("row"), or divided by a given device
    float32 scale [1]. out: y's buffer; out_h: h's, which may be x or residual itself.
    """
    if stream is not None:
        return _on(stream, rms_norm, x, weight, residual, eps, out_dtype, scale, out, out_h)
    dtype = x.dtype
    dt = _T16.get(dtype)
    if dt is None:
        raise TypeError("x must be bfloat16 or float16")
    xs = _matrix("x", x)
    (m, n), dev = x.shape, x.device
    wd = weight.dtype
    if wd != dtype and wd != torch.float32:
        raise TypeError("weight must be of x's type or float32")
    _flat("weight", weight, wd, (n,), dev)
    rs = hs = hp = 0
    h = x
    if residual is not None:
        _like("residual", residual, x)
        rs = _matrix("residual", residual)
        if out_h is None:
            h = _new_like(x)
            hs = n
        else:
            h = out_h
            _like("out_h", h, x)
            hs = _matrix("out_h", h)
        hp = h.data_ptr()
    elif out_h is not None:
        raise ValueError("out_h goes with a residual")
    ws = s = None
    if out_dtype is None or out_dtype == dtype:
        if scale is not None:
            raise ValueError("scale goes with an fp8 out_dtype")
        out_dtype, od, mode = dtype, dt, _PLAIN
    else:
        od = _T8.get(out_dtype)
        if od is None:
            raise TypeError("out_dtype must be x's type, float8_e4m3fn or float8_e5m2")
        if scale is None or isinstance(scale, str):
            if scale not in (None, "tensor", "row"):
                raise ValueError("scale must be 'tensor', 'row' or a device float32 tensor of one value")
            mode = _ROW if scale == "row" else _TENSOR
            s = torch.empty(m if mode == _ROW else 1, dtype=torch.float32, device=dev)
            if mode == _TENSOR:
                ws = torch.empty(_NORM_WORKSPACE, dtype=torch.uint8, device=dev)
        else:
            mode, s = _GIVEN, scale
            if s.dtype != torch.float32 or s.numel() != 1 or s.device != dev:
                raise ValueError("scale must be 'tensor', 'row' or a device float32 tensor of one value")
    y = _new_like(x) if out is None and mode == _PLAIN else _out(out, out_dtype, (m, n), dev)
    rstd = torch.empty(m, dtype=torch.float32, device=dev)
    _call(_lib.gg_rms_norm, dev, (dt, dt if wd == dtype else _FP32, od, mode, m, n, eps, x.data_ptr(), xs, _ptr(residual), rs,
                                  weight.data_ptr(), hp, hs, y.data_ptr(), rstd.data_ptr(), _ptr(s), _ptr(ws)))
    return NormOutput(y, h, rstd, s)


def rms_norm_backward(grad_y, h, weight, rstd, grad_h=None, out=None, stream: Optional[int] = None):
    """(grad_x, grad_weight) of rms_norm from its h and rstd (gg_rms_norm_backward). grad_x is the gradient
    of x and of residual; grad_h, the gradient that reaches h past the norm, is added to it. grad_y and
    grad_h are of h's type (an fp8 y is differentiated as if it were not rounded)."""
    if stream is not None:
        return _on(stream, rms_norm_backward, grad_y, h, weight, rstd, grad_h, out)
    dtype = h.dtype
    dt = _T16.get(dtype)
    if dt is None:
        raise TypeError("h must be bfloat16 or float16")
    hs = _matrix("h", h)
    (m, n), dev = h.shape, h.device
    _like("grad_y", grad_y, h)
    gs, ghs = _matrix("grad_y", grad_y), 0
    if grad_h is not None:
        _like("grad_h", grad_h, h)
        ghs = _matrix("grad_h", grad_h)
    wd = weight.dtype
    if wd != dtype and wd != torch.float32:
        raise TypeError("weight must be of h's type or float32")
    _flat("weight", weight, wd, (n,), dev)
    _flat("rstd", rstd, torch.float32, (m,), dev)
    gx = _new_like(h) if out is None else _out(out, dtype, (m, n), dev)
    gw = torch.empty_like(weight)
    need = _lib.gg_rms_norm_backward_workspace(m, n)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    _call(_lib.gg_rms_norm_backward, dev, (dt, dt if wd == dtype else _FP32, m, n, grad_y.data_ptr(), gs, h.data_ptr(), hs,
                                           weight.data_ptr(), rstd.data_ptr(), _ptr(grad_h), ghs, gx.data_ptr(),
                                           gw.data_ptr(), _ptr(ws), need))
    return gx, gw


# ---- router ----


class Routing(NamedTuple):
    """What route gives, and what dispatch, combine and the backward functions take of it.

    experts [T, k] int32 (-1: none), weights [T, k] float32, counts [E] int64 (device group sizes of the
    grouped GEMMs), offs [E + 1] int64 (their group_offs), rows [T, k] int32 (row of each pair in expert
    order, -1: none), lse [T] float32, slope [E] float32 and loss [] float32 (None without balance).
    """
    experts: "torch.Tensor"
    weights: "torch.Tensor"
    counts: "torch.Tensor"
    offs: "torch.Tensor"
    rows: "torch.Tensor"
    lse: "torch.Tensor"
    slope: "Optional[torch.Tensor]" = None
    loss: "Optional[torch.Tensor]" = None
    renormalize: bool = True


def _logits(logits):
    dt = _FP32 if logits.dtype == torch.float32 else _T16.get(logits.dtype)
    if dt is None:
        raise TypeError("logits must be float32, bfloat16 or float16")
    return dt, _matrix("logits", logits)


def route(logits, top_k: int, mask=None, renormalize: bool = True, balance: bool = False,
          stream: Optional[int] = None) -> Routing:
    """Top-k routing of logits [T, E] (gg_route): the top_k largest logits of each token in descending order
    (equal ones by the lower index), their softmax weights (divided by their sum with renormalize), the rows
    of each expert and of each pair, and with balance the loss E * sum(f * P) over the tokens that take part.
    mask [T] bool: False = the token takes no part (padding); its logits are not looked at."""
    if stream is not None:
        return _on(stream, route, logits, top_k, mask, renormalize, balance)
    dt, stride = _logits(logits)
    (t, e), dev = logits.shape, logits.device
    if mask is not None:
        _flat("mask", mask, torch.bool, (t,), dev)
    if not 1 <= top_k <= e:
        raise ValueError("top_k must be in 1 .. E")
    experts = torch.empty((t, top_k), dtype=torch.int32, device=dev)
    rows = torch.empty_like(experts)
    weights = torch.empty_like(experts, dtype=torch.float32)
    counts = torch.empty(e, dtype=torch.int64, device=dev)
    offs = torch.empty(e + 1, dtype=torch.int64, device=dev)
    lse = torch.empty(t, dtype=torch.float32, device=dev)
    slope = loss = ws = None
    if balance:
        slope = torch.empty(e, dtype=torch.float32, device=dev)
        loss = torch.empty((), dtype=torch.float32, device=dev)
    need = _lib.gg_route_workspace(t, e, top_k)
    if need:
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
    _call(_lib.gg_route, dev, (dt, t, e, top_k, int(renormalize), logits.data_ptr(), stride, _ptr(mask), experts.data_ptr(),
                               weights.data_ptr(), counts.data_ptr(), offs.data_ptr(), rows.data_ptr(), lse.data_ptr(),
                               _ptr(loss), _ptr(slope), _ptr(ws), need))
    return Routing(experts, weights, counts, offs, rows, lse, slope, loss, bool(renormalize))


def route_backward(logits, routing: Routing, grad_weights=None, grad_loss=None, out=None, stream: Optional[int] = None):
    """Gradient of the logits, in their type, from the gradients of routing.weights [T, k] float32 and of
    routing.loss (a device float32 tensor of one value), either of them None (gg_route_backward)."""
    if stream is not None:
        return _on(stream, route_backward, logits, routing, grad_weights, grad_loss, out)
    dt, stride = _logits(logits)
    (t, e), dev = logits.shape, logits.device
    r = routing
    k = r.experts.shape[1]
    _flat("routing.experts", r.experts, torch.int32, (t, k), dev)
    _flat("routing.weights", r.weights, torch.float32, (t, k), dev)
    _flat("routing.lse", r.lse, torch.float32, (t,), dev)
    if grad_weights is not None:
        _flat("grad_weights", grad_weights, torch.float32, (t, k), dev)
    if grad_loss is not None:
        if r.slope is None:
            raise ValueError("grad_loss goes with a routing that has a balance loss")
        _flat("routing.slope", r.slope, torch.float32, (e,), dev)
        if grad_loss.dtype != torch.float32 or grad_loss.numel() != 1 or grad_loss.device != dev:
            raise ValueError("grad_loss must be a device float32 tensor of one value")
    g = _new_like(logits) if out is None else _out(out, logits.dtype, (t, e), dev)
    _call(_lib.gg_route_backward, dev, (dt, t, e, k, int(r.renormalize), logits.data_ptr(), stride, r.experts.data_ptr(),
                                        r.weights.data_ptr(), r.lse.data_ptr(), _ptr(grad_weights), _ptr(grad_loss),
                                        0 if grad_loss is None else r.slope.data_ptr(), g.data_ptr()))
    return g


# ---- rows of the experts ----


def _rows(routing: Routing, dev):
    rows = routing.rows
    if rows.dim() != 2:
        raise ValueError("routing.rows must be a matrix")
    t, k = rows.shape
    _flat("routing.rows", rows, torch.int32, (t, k), dev)
    return rows, t, k


def _offs(routing: Routing, dev):
    offs = routing.offs
    _flat("routing.offs", offs, torch.int64, (offs.numel(),), dev)
    if offs.numel() < 1:
        raise ValueError("routing.offs must hold E + 1 entries")
    return offs


def dispatch(x, routing: Routing, out=None, stream: Optional[int] = None):
    """xs [T * k, H]: row routing.rows[t, s] is x[t]; rows past the last expert's are zero (gg_dispatch). x:
    [T, H] of any type of 1, 2 or 4 bytes, rows contiguous. xs with routing.counts is what grouped_gemm takes."""
    if stream is not None:
        return _on(stream, dispatch, x, routing, out)
    stride, dev = _matrix("x", x), x.device
    rows, t, k = _rows(routing, dev)
    offs = _offs(routing, dev)
    if x.shape[0] != t:
        raise ValueError("x must have a row for each token of the routing")
    n = x.shape[1]
    if x.element_size() not in (1, 2, 4):
        raise TypeError("x must be of a type of 1, 2 or 4 bytes")
    xs = _out(out, x.dtype, (t * k, n), dev)
    _call(_lib.gg_dispatch, dev, (x.element_size(), t, k, n, offs.numel() - 1, x.data_ptr(), stride, rows.data_ptr(),
                                  offs.data_ptr(), xs.data_ptr()))
    return xs


def _pairs(name: str, y, t: int, k: int):
    if y.dtype not in _T16:
        raise TypeError(f"{name} must be bfloat16 or float16")
    if y.dim() != 2 or not y.is_cuda or y.shape[0] != t * k or not y.is_contiguous():
        raise ValueError(f"{name} must be a contiguous device matrix with a row for each (token, slot) pair of the routing")
    return y.shape[1]


def dispatch_backward(grad_xs, routing: Routing, out=None, stream: Optional[int] = None):
    """grad_x [T, H]: the sum of each token's rows of grad_xs [T * k, H] (gg_dispatch_backward)."""
    if stream is not None:
        return _on(stream, dispatch_backward, grad_xs, routing, out)
    dev = grad_xs.device
    rows, t, k = _rows(routing, dev)
    n = _pairs("grad_xs", grad_xs, t, k)
    gx = _out(out, grad_xs.dtype, (t, n), dev)
    _call(_lib.gg_dispatch_backward, dev, (_T16[grad_xs.dtype], t, k, n, grad_xs.data_ptr(), rows.data_ptr(), gx.data_ptr()))
    return gx


def combine(y, routing: Routing, out=None, stream: Optional[int] = None):
    """out [T, H]: the sum of each token's rows of y [T * k, H], times routing.weights (gg_combine)."""
    if stream is not None:
        return _on(stream, combine, y, routing, out)
    dev = y.device
    rows, t, k = _rows(routing, dev)
    n = _pairs("y", y, t, k)
    _flat("routing.weights", routing.weights, torch.float32, (t, k), dev)
    o = _out(out, y.dtype, (t, n), dev)
    _call(_lib.gg_combine, dev, (_T16[y.dtype], t, k, n, y.data_ptr(), rows.data_ptr(), routing.weights.data_ptr(),
                                 o.data_ptr()))
    return o


def combine_backward(grad_out, y, routing: Routing, out=None, stream: Optional[int] = None):
    """(grad_y [T * k, H], grad_weights [T, k] float32) of combine (gg_combine_backward). grad_out: [T, H] of
    y's type, rows contiguous. Rows of grad_y past the last expert's are zero."""
    if stream is not None:
        return _on(stream, combine_backward, grad_out, y, routing, out)
    dev = y.device
    rows, t, k = _rows(routing, dev)
    offs = _offs(routing, dev)
    n = _pairs("y", y, t, k)
    _flat("routing.weights", routing.weights, torch.float32, (t, k), dev)
    if grad_out.dtype != y.dtype or grad_out.device != dev or tuple(grad_out.shape) != (t, n):
        raise ValueError("grad_out must be [T, H] of y's type")
    stride = _matrix("grad_out", grad_out)
    gy = _out(out, y.dtype, (t * k, n), dev)
    gw = torch.empty((t, k), dtype=torch.float32, device=dev)
    _call(_lib.gg_combine_backward, dev, (_T16[y.dtype], t, k, n, offs.numel() - 1, grad_out.data_ptr(), stride, y.data_ptr(),
                                          rows.data_ptr(), offs.data_ptr(), routing.weights.data_ptr(), gy.data_ptr(),
                                          gw.data_ptr()))
    return gy, gw


# ---- 4-bit weights ----


class W4Weights(NamedTuple):
    """Weights [B, N, K] in 4 bits as gg_gemm_w4 reads them: packed uint8 [B, ceil(N / 16), ceil(K / 128), 64,
    16], scales [B, ceil(N / 16), K / group, 16], zeros uint8 of the same shape or None (8)."""
    packed: "torch.Tensor"
    scales: "torch.Tensor"
    zeros: "Optional[torch.Tensor]"
    n: int
    k: int
    group: int


def pack_w4(q, scales, zeros=None) -> W4Weights:
    """Lays out weights scale * (q - zero) once: q [B, N, K] uint8 in 0..15, scales [B, N, K / group] bf16 or
    fp16, zeros [B, N, K / group] uint8 in 0..15 or None (8 everywhere). Any device."""
    if q.dim() != 3 or q.dtype != torch.uint8:
        raise ValueError("q must be uint8 [B, N, K]")
    b, n, k = q.shape
    if scales.dtype not in _T16 or scales.dim() != 3 or scales.shape[:2] != q.shape[:2] or scales.shape[2] < 1 \
            or k % scales.shape[2] != 0:
        raise ValueError("scales must be bfloat16 or float16 [B, N, K / group]")
    group = k // scales.shape[2]
    if group not in (32, 64, 128):
        raise ValueError("group must be 32, 64 or 128")
    if zeros is not None and (zeros.dtype != torch.uint8 or zeros.shape != scales.shape):
        raise ValueError("zeros must be uint8 of the scales' shape")
    nt, kt = (n + 15) // 16, (k + 127) // 128
    packed = torch.empty((b, nt, kt, 64, 16), dtype=torch.uint8, device=q.device)
    for i in range(b):  # one matrix at a time: the layers' weights may fill the card
        if bool((q[i] > 15).any()):  # would reach into the weight that shares its byte
            raise ValueError("q must be uint8 [B, N, K] in 0..15")
        full = torch.zeros((nt * 16, kt * 128), dtype=torch.uint8, device=q.device)
        full[:n, :k] = q[i]
        # rows r, k = 128 c + 32 j + 8 a + 2 p + o -> piece 16 a + r, word j, half o, nibble p
        v = full.view(nt, 16, kt, 4, 4, 4, 2).permute(0, 2, 4, 1, 3, 6, 5).reshape(nt, kt, 64, 16, 2)
        packed[i] = v[..., 0] | (v[..., 1] << 4)

    def tiles(s):
        full = torch.zeros((b, nt * 16, s.shape[2]), dtype=s.dtype, device=s.device)
        full[:, :n] = s
        return full.view(b, nt, 16, -1).transpose(2, 3).contiguous()

    return W4Weights(packed, tiles(scales), None if zeros is None else tiles(zeros), n, k, group)


def quantize_w4(w, group: int = 128, zeros: bool = False) -> W4Weights:
    """4-bit form of weights [B, N, K] (bf16 or fp16), one scale for each `group` consecutive k of a row:
    symmetric (largest |w| at 7.5 steps from the zero at 8), or with a zero point between least and greatest."""
    if w.dim() != 3 or w.dtype not in _T16:
        raise ValueError("w must be bfloat16 or float16 [B, N, K]")
    b, n, k = w.shape
    if group not in (32, 64, 128) or k % group != 0:
        raise ValueError("group must be 32, 64 or 128 and divide K")
    q = torch.empty((b, n, k), dtype=torch.uint8, device=w.device)
    s = torch.empty((b, n, k // group), dtype=w.dtype, device=w.device)
    z = torch.empty((b, n, k // group), dtype=torch.uint8, device=w.device) if zeros else None
    for i in range(b):
        v = w[i].float().view(n, k // group, group)
        if zeros:
            lo, hi = v.amin(2).clamp(max=0.0), v.amax(2).clamp(min=0.0)
            step = ((hi - lo) / 15).to(w.dtype)
        else:
            step = (v.abs().amax(2) / 7.5).to(w.dtype)
        step = torch.where(step > 0, step, torch.ones_like(step))  # a group of zeros
        at = (-lo / step.float()).round().clamp(0, 15) if zeros else torch.full_like(step, 8, dtype=torch.float32)
        q[i] = (v / step.float()[:, :, None] + at[:, :, None]).round().clamp(0, 15).to(torch.uint8).view(n, k)
        s[i] = step
        if zeros:
            z[i] = at.to(torch.uint8)
    return pack_w4(q, s, z)


def grouped_gemm_w4(x, w: W4Weights, group_m, out=None, stream: Optional[int] = None, group_offs=None):
    """out [sum(M), N] = x[rows of g] @ w[g]^T for 4-bit weights (gg_gemm_w4), x bf16 or fp16 [sum(M), K] of
    the scales' type. group_m as in grouped_gemm: a host sequence of row counts, or a device int64 tensor [B]
    that is never read on the host (with optional device offsets); a device group that does not lie inside x
    gets no work, and rows of no group are not written. For groups of few rows: every 16 or 32 rows of a group read
    its weights once."""
    if stream is not None:
        return _on(stream, grouped_gemm_w4, x, w, group_m, out, None, group_offs)
    dt = _T16.get(x.dtype)
    if dt is None:
        raise TypeError("x must be bfloat16 or float16")
    dev = x.device
    packed, scales, zeros, n, k, group = w
    b, nt = packed.shape[0], (n + 15) // 16
    if scales.dtype != x.dtype:
        raise TypeError("the scales must be of x's type")
    _flat("w.packed", packed, torch.uint8, (b, nt, (k + 127) // 128, 64, 16), dev)
    shape = (b, nt, k // group, 16)
    _flat("w.scales", scales, x.dtype, shape, dev)
    if zeros is not None:
        _flat("w.zeros", zeros, torch.uint8, shape, dev)
    if x.dim() != 2 or not x.is_cuda or x.shape[1] != k or not x.is_contiguous():
        raise ValueError("x must be a contiguous device matrix with K columns")
    m = x.shape[0]
    if not _device_sizes(group_m, group_offs, b):
        if len(group_m) != b or any(r < 0 for r in group_m) or sum(group_m) != m:
            raise ValueError("shape mismatch between x, w and group_m")
        group_m = torch.tensor(list(group_m), dtype=torch.int64, device=dev)
    elif group_m.device != dev or (group_offs is not None and group_offs.device != dev):
        raise ValueError("group sizes must be on x's device")
    o = _out(out, x.dtype, (m, n), dev)
    _call(_lib.gg_gemm_w4, dev, (dt, b, m, n, k, group, group_m.data_ptr(), _ptr(group_offs), x.data_ptr(), packed.data_ptr(),
                                 scales.data_ptr(), _ptr(zeros), o.data_ptr()))
    return o
