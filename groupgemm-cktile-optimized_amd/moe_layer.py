"""The operators around the grouped GEMM in a mixture-of-experts layer, for torch tensors, over the C
ABI in include/gg_moe_layer.h: RMS norm and layer norm with the residual's addition and an 8-bit output,
gated activation, rows of int8, router with balance loss, dispatch and combine of the experts' rows,
grouped products with 4-bit weights and in 8-bit integers.

Every function enqueues its kernels on the current stream of its tensors' device, or on `stream` (a
raw hipStream_t handle), and returns without waiting (but grouped_gemm_w4 and grouped_gemm_i8 with host
group sizes, which copy them to the device and wait for that). Outputs and workspaces come from torch's allocator, from
the memory of the stream that the kernels run on. With `stream`, the caller orders that stream after
whatever wrote the inputs, and what reads the outputs on another stream after it; the allocator is told
of both streams' uses, so a tensor may be dropped before the work is done.
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import GG_ERR_UNSUPPORTED, GG_OK, DType, GGError, _device_sizes, load_library

_T16 = {torch.bfloat16: int(DType.BF16), torch.float16: int(DType.FP16)}
_T8 = {torch.float8_e4m3fn: int(DType.FP8_E4M3), torch.float8_e5m2: int(DType.FP8_E5M2)}
_FP32, _INT8 = 4, 5  # GG_DTYPE_FP32, GG_DTYPE_INT8
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
    ([1], or [M] for one a row) of an 8-bit y, which stands for y * scale, else None."""
    y: "torch.Tensor"
    h: "torch.Tensor"
    rstd: "torch.Tensor"
    scale: "Optional[torch.Tensor]"


class LayerNormOutput(NamedTuple):
    """layer_norm's outputs: y; h = x + residual (x itself without one); mean and rstd [M] float32; scale float32
    ([1], or [M] for one a row) of an 8-bit y, which stands for y * scale, else None."""
    y: "torch.Tensor"
    h: "torch.Tensor"
    mean: "torch.Tensor"
    rstd: "torch.Tensor"
    scale: "Optional[torch.Tensor]"


def _norm(center: bool, x, weight, bias, residual, eps, out_dtype, scale, out, out_h):
    """(y, h, mean, rstd, scale) of either norm."""
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
    if bias is not None:
        _flat("bias", bias, wd, (n,), dev)
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
            raise ValueError("scale goes with an 8-bit out_dtype")
        out_dtype, od, mode = dtype, dt, _PLAIN
    else:
        od = _T8.get(out_dtype)
        if od is None and out_dtype != torch.int8:
            raise TypeError("out_dtype must be x's type, float8_e4m3fn, float8_e5m2 or int8")
        if od is None:
            if not isinstance(scale, str) or scale != "row":
                raise ValueError("int8 rows have a scale each: scale must be 'row'")
            od, mode, s = _INT8, _ROW, torch.empty(m, dtype=torch.float32, device=dev)
        elif scale is None or isinstance(scale, str):
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
    wt = dt if wd == dtype else _FP32
    if not center:
        _call(_lib.gg_rms_norm, dev, (dt, wt, od, mode, m, n, eps, x.data_ptr(), xs, _ptr(residual), rs, weight.data_ptr(),
                                      hp, hs, y.data_ptr(), rstd.data_ptr(), _ptr(s), _ptr(ws)))
        return y, h, None, rstd, s
    mean = torch.empty_like(rstd)
    _call(_lib.gg_layer_norm, dev, (dt, wt, od, mode, m, n, eps, x.data_ptr(), xs, _ptr(residual), rs, weight.data_ptr(), _ptr(bias),
                                    hp, hs, y.data_ptr(), mean.data_ptr(), rstd.data_ptr(), _ptr(s), _ptr(ws)))
    return y, h, mean, rstd, s


def rms_norm(x, weight, residual=None, eps: float = 1e-6, out_dtype=None, scale=None, out=None, out_h=None,
             stream: Optional[int] = None) -> NormOutput:
    """y = h * rsqrt(mean(h^2) + eps) * weight over the rows of h = x + residual (gg_rms_norm).

    x, residual: [M, H] bf16 or fp16, rows contiguous at any stride; weight [H] of x's type or float32.
    out_dtype float8_e4m3fn or float8_e5m2 gives an fp8 y: with one scale for the tensor (scale=None or
    "tensor": the x_scale of grouped_gemm_fp8), one for each row ("row"), or divided by a given device
    float32 scale [1]; int8 with scale="row" the rows and scales of grouped_gemm_i8. out: y's buffer; out_h:
    h's, which may be x or residual itself.
    """
    if stream is not None:
        return _on(stream, rms_norm, x, weight, residual, eps, out_dtype, scale, out, out_h)
    y, h, _, rstd, s = _norm(False, x, weight, None, residual, eps, out_dtype, scale, out, out_h)
    return NormOutput(y, h, rstd, s)


def layer_norm(x, weight, bias=None, residual=None, eps: float = 1e-5, out_dtype=None, scale=None, out=None, out_h=None,
               stream: Optional[int] = None) -> LayerNormOutput:
    """y = (h - mean) * rstd * weight + bias over the rows of h = x + residual, rstd = rsqrt(mean((h - mean)^2) + eps)
    (gg_layer_norm). bias [H] of weight's type or None; everything else as in rms_norm."""
    if stream is not None:
        return _on(stream, layer_norm, x, weight, bias, residual, eps, out_dtype, scale, out, out_h)
    return LayerNormOutput(*_norm(True, x, weight, bias, residual, eps, out_dtype, scale, out, out_h))


def _norm_back(center: bool, grad_y, h, weight, mean, rstd, grad_h, out):
    """(grad_x, grad_weight, grad_bias) of either norm."""
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
    if center:
        _flat("mean", mean, torch.float32, (m,), dev)
    gx = _new_like(h) if out is None else _out(out, dtype, (m, n), dev)
    gw = torch.empty_like(weight)
    gb = torch.empty_like(weight) if center else None
    need = (_lib.gg_layer_norm_backward_workspace if center else _lib.gg_rms_norm_backward_workspace)(m, n)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    wt = dt if wd == dtype else _FP32
    if center:
        _call(_lib.gg_layer_norm_backward, dev, (dt, wt, m, n, grad_y.data_ptr(), gs, h.data_ptr(), hs, weight.data_ptr(),
                                                 mean.data_ptr(), rstd.data_ptr(), _ptr(grad_h), ghs, gx.data_ptr(),
                                                 gw.data_ptr(), gb.data_ptr(), _ptr(ws), need))
    else:
        _call(_lib.gg_rms_norm_backward, dev, (dt, wt, m, n, grad_y.data_ptr(), gs, h.data_ptr(), hs, weight.data_ptr(),
                                               rstd.data_ptr(), _ptr(grad_h), ghs, gx.data_ptr(), gw.data_ptr(), _ptr(ws), need))
    return gx, gw, gb


def rms_norm_backward(grad_y, h, weight, rstd, grad_h=None, out=None, stream: Optional[int] = None):
    """(grad_x, grad_weight) of rms_norm from its h and rstd (gg_rms_norm_backward). grad_x is the gradient
    of x and of residual; grad_h, the gradient that reaches h past the norm, is added to it. grad_y and
    grad_h are of h's type (an 8-bit y is differentiated as if it were not rounded)."""
    if stream is not None:
        return _on(stream, rms_norm_backward, grad_y, h, weight, rstd, grad_h, out)
    gx, gw, _ = _norm_back(False, grad_y, h, weight, None, rstd, grad_h, out)
    return gx, gw


def layer_norm_backward(grad_y, h, weight, mean, rstd, grad_h=None, out=None, stream: Optional[int] = None):
    """(grad_x, grad_weight, grad_bias) of layer_norm from its h, mean and rstd (gg_layer_norm_backward); as
    rms_norm_backward. grad_bias is of weight's type, whether there was a bias or not."""
    if stream is not None:
        return _on(stream, layer_norm_backward, grad_y, h, weight, mean, rstd, grad_h, out)
    return _norm_back(True, grad_y, h, weight, mean, rstd, grad_h, out)


# ---- gated activation, rows of int8 ----


class ScaledRows(NamedTuple):
    """Rows y [M, N] and, where they are int8, scale [M] float32: row i stands for y[i] * scale[i]. Else scale is None."""
    y: "torch.Tensor"
    scale: "Optional[torch.Tensor]"


def _gates(gu):
    dt = _T16.get(gu.dtype)
    if dt is None:
        raise TypeError("gu must be bfloat16 or float16")
    stride = _matrix("gu", gu)
    if gu.shape[1] % 2:
        raise ValueError("gu must hold as many gates as ups")
    return dt, stride, gu.shape[1] // 2


def silu_product(gu, out_dtype=None, out=None, stream: Optional[int] = None) -> ScaledRows:
    """y = silu(gate) * up of rows gu [M, 2 N] that hold N gates and then N ups, rows contiguous at any stride
    (gg_silu_product). y is of gu's type, or with out_dtype=int8 rounded to int8 rows with a scale each, as
    grouped_gemm_i8 takes them."""
    if stream is not None:
        return _on(stream, silu_product, gu, out_dtype, out)
    dt, stride, n = _gates(gu)
    m, dev = gu.shape[0], gu.device
    if out_dtype is None or out_dtype == gu.dtype:
        y, s, od = _out(out, gu.dtype, (m, n), dev), None, dt
    elif out_dtype == torch.int8:
        y, s, od = _out(out, torch.int8, (m, n), dev), torch.empty(m, dtype=torch.float32, device=dev), _INT8
    else:
        raise TypeError("out_dtype must be gu's type or int8")
    _call(_lib.gg_silu_product, dev, (dt, od, m, n, gu.data_ptr(), stride, y.data_ptr(), _ptr(s)))
    return ScaledRows(y, s)


def silu_product_backward(grad_y, gu, out=None, stream: Optional[int] = None):
    """grad_gu [M, 2 N] of silu_product from grad_y [M, N] of gu's type (gg_silu_product_backward; an int8 y is
    differentiated as if it were not rounded). out may be a contiguous gu itself."""
    if stream is not None:
        return _on(stream, silu_product_backward, grad_y, gu, out)
    dt, stride, n = _gates(gu)
    m, dev = gu.shape[0], gu.device
    if grad_y.dtype != gu.dtype or grad_y.device != dev or tuple(grad_y.shape) != (m, n):
        raise ValueError("grad_y must be [M, N] of gu's type")
    gs = _matrix("grad_y", grad_y)
    o = _new_like(gu) if out is None else _out(out, gu.dtype, (m, 2 * n), dev)
    _call(_lib.gg_silu_product_backward, dev, (dt, m, n, grad_y.data_ptr(), gs, gu.data_ptr(), stride, o.data_ptr()))
    return o


def quantize_rows(x, out=None, stream: Optional[int] = None) -> ScaledRows:
    """int8 rows of x [M, N] (bf16 or fp16, rows contiguous at any stride) and a scale for each (gg_quantize_rows):
    scale = max |x| / 127 (1 where that is zero or subnormal), y = x / scale rounded to the nearest, halves to even. A row with
    a NaN or an infinity has that for a scale and holds zeros. N at most 32768."""
    if stream is not None:
        return _on(stream, quantize_rows, x, out)
    dt = _T16.get(x.dtype)
    if dt is None:
        raise TypeError("x must be bfloat16 or float16")
    stride, dev = _matrix("x", x), x.device
    m, n = x.shape
    y, s = _out(out, torch.int8, (m, n), dev), torch.empty(m, dtype=torch.float32, device=dev)
    _call(_lib.gg_quantize_rows, dev, (dt, m, n, x.data_ptr(), stride, y.data_ptr(), s.data_ptr()))
    return ScaledRows(y, s)


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


def dispatch_scaled(x, scale, routing: Routing, out=None, stream: Optional[int] = None) -> ScaledRows:
    """dispatch of rows that have a scale each (gg_dispatch_scaled): x [T, H] and scale [T] float32, as layer_norm,
    rms_norm and quantize_rows give them, to xs [T * k, H] and its scales [T * k]; those of the zeroed rows are 0."""
    if stream is not None:
        return _on(stream, dispatch_scaled, x, scale, routing, out)
    stride, dev = _matrix("x", x), x.device
    rows, t, k = _rows(routing, dev)
    offs = _offs(routing, dev)
    if x.shape[0] != t:
        raise ValueError("x must have a row for each token of the routing")
    _flat("scale", scale, torch.float32, (t,), dev)
    n = x.shape[1]
    if x.element_size() not in (1, 2, 4):
        raise TypeError("x must be of a type of 1, 2 or 4 bytes")
    xs = _out(out, x.dtype, (t * k, n), dev)
    s = torch.empty(t * k, dtype=torch.float32, device=dev)
    _call(_lib.gg_dispatch_scaled, dev, (x.element_size(), t, k, n, offs.numel() - 1, x.data_ptr(), stride, scale.data_ptr(),
                                         rows.data_ptr(), offs.data_ptr(), xs.data_ptr(), s.data_ptr()))
    return ScaledRows(xs, s)


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


# ---- 8-bit integers ----


class I8Weights(NamedTuple):
    """Weights [B, N, K] in int8 and a float32 scale for each output channel, scales [B, N]: w[b, n] * scales[b, n]."""
    w: "torch.Tensor"
    scales: "torch.Tensor"


def quantize_i8(w) -> I8Weights:
    """int8 form of weights [B, N, K] (bf16, fp16 or float32), one scale for each output channel: max |w| / 127 (1 for a
    channel of zeros), values rounded to the nearest. A channel with a NaN or an infinity has that for a scale and holds
    zeros, so that what is multiplied by it is NaN. Any device."""
    if w.dim() != 3 or w.dtype not in (*_T16, torch.float32):
        raise ValueError("w must be bfloat16, float16 or float32 [B, N, K]")
    q = torch.empty(w.shape, dtype=torch.int8, device=w.device)
    s = torch.empty(w.shape[:2], dtype=torch.float32, device=w.device)
    for i in range(w.shape[0]):  # one matrix at a time: the layers' weights may fill the card
        v = w[i].detach().float()
        top = v.abs().amax(1) / 127
        s[i] = torch.where(top == 0, torch.ones_like(top), top)
        q[i] = torch.where(top.isfinite()[:, None], v / s[i][:, None], torch.zeros_like(v)).round().clamp(-127, 127).to(torch.int8)
    return I8Weights(q, s)


def grouped_gemm_i8(x, w: I8Weights, group_m, x_scale=None, out_dtype=None, out=None, stream: Optional[int] = None,
                    group_offs=None):
    """out [sum(M), N] = x[rows of g] @ w[g]^T in 8-bit integers (gg_gemm_i8): x int8 [sum(M), K] with x_scale [sum(M)]
    float32, the ScaledRows of layer_norm, silu_product, quantize_rows or dispatch_scaled, to out_dtype (bfloat16 if None,
    or float16), K below 131072; or x bfloat16 or float16, whose rows are first rounded by quantize_rows, to x's type, K at
    most 32768. group_m as in grouped_gemm: a host sequence of row counts, or a device int64 tensor [B] that is never read
    on the host (with optional device offsets); a device group that does not lie inside x gets no work, and rows of no group
    are not written. For any number of rows. No backward pass: train in 16 bits."""
    if stream is not None:
        return _on(stream, grouped_gemm_i8, x, w, group_m, x_scale, out_dtype, out, None, group_offs)
    q, scales = w
    if q.dim() != 3 or q.dtype != torch.int8 or not q.is_contiguous():
        raise ValueError("w must be contiguous int8 [B, N, K] with its scales")
    b, n, k = q.shape
    dev = x.device
    if x.dim() != 2 or not x.is_cuda or x.shape[1] != k:
        raise ValueError("x must be a device matrix with K columns")
    if x.dtype == torch.int8:
        if x_scale is None:
            raise ValueError("int8 x needs x_scale, a scale for each row")
        if out_dtype is None:
            out_dtype = torch.bfloat16
        elif out_dtype not in _T16:
            raise TypeError("out_dtype must be bfloat16 or float16")
        if not x.is_contiguous():
            raise ValueError("int8 x must be contiguous")
    elif x.dtype in _T16:
        if x_scale is not None or out_dtype not in (None, x.dtype):
            raise ValueError("x_scale and out_dtype go with an int8 x")
        if k > 32768:  # quantize_rows' limit, in this call's words
            raise GGError(GG_ERR_UNSUPPORTED, "K must be at most 32768 for x of 16 bits; int8 x may have K below 131072")
        out_dtype = x.dtype
    else:
        raise TypeError("x must be int8, bfloat16 or float16")
    _flat("w.scales", scales, torch.float32, (b, n), dev)
    if q.device != dev:
        raise ValueError("w must be on x's device")
    m = x.shape[0]
    if not _device_sizes(group_m, group_offs, b):
        if len(group_m) != b or any(r < 0 for r in group_m) or sum(group_m) != m:
            raise ValueError("shape mismatch between x, w and group_m")
        group_m = torch.tensor(list(group_m), dtype=torch.int64, device=dev)
    elif group_m.device != dev or (group_offs is not None and group_offs.device != dev):
        raise ValueError("group sizes must be on x's device")
    if x.dtype != torch.int8:
        x, x_scale = quantize_rows(x)
    else:
        _flat("x_scale", x_scale, torch.float32, (m,), dev)
    o = _out(out, out_dtype, (m, n), dev)
    need = _lib.gg_gemm_i8_workspace(b)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    _call(_lib.gg_gemm_i8, dev, (_T16[out_dtype], b, m, n, k, group_m.data_ptr(), _ptr(group_offs), x.data_ptr(), q.data_ptr(),
                                 x_scale.data_ptr(), scales.data_ptr(), o.data_ptr(), ws.data_ptr(), need))
    return o
