"""One mixture-of-experts layer on this package's operators: a training step, an fp8 forward pass and a
decode step on 4-bit experts.

    h = x + residual;  y = rms_norm(h);  out = sum over a token's experts of weight * expert(y)
    expert(y) = down(silu(gate(y)) * up(y))

    python3 groupgemm-cktile-optimized_amd/moe_example.py [--tokens 4096] [--hidden 2048] [--inner 1408] [--experts 32]
                                                          [--top-k 4] [--decode 8]

prints what each pass takes, and how far the fp8 and 4-bit passes are from the 16-bit one.
"""
from __future__ import annotations

import argparse
import os
import sys
import time

import torch

if __package__:
    from . import (combine, combine_backward, dispatch, dispatch_backward, grouped_gemm, grouped_gemm_dgrad, grouped_gemm_fp8,
                   grouped_gemm_w4, grouped_gemm_wgrad, quantize_w4, rms_norm, rms_norm_backward, route, route_backward)
else:  # run as a file
    sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    import __graft_entry__

    _gg = __graft_entry__.load_package()
    combine, combine_backward, dispatch, dispatch_backward = _gg.combine, _gg.combine_backward, _gg.dispatch, _gg.dispatch_backward
    grouped_gemm, grouped_gemm_dgrad, grouped_gemm_wgrad = _gg.grouped_gemm, _gg.grouped_gemm_dgrad, _gg.grouped_gemm_wgrad
    grouped_gemm_fp8, grouped_gemm_w4, quantize_w4 = _gg.grouped_gemm_fp8, _gg.grouped_gemm_w4, _gg.quantize_w4
    rms_norm, rms_norm_backward, route, route_backward = _gg.rms_norm, _gg.rms_norm_backward, _gg.route, _gg.route_backward


def _silu_product(gu):
    gate, up = gu.float().chunk(2, dim=1)
    return (gate * torch.sigmoid(gate) * up).to(gu.dtype)


def _silu_product_backward(gu, grad):
    gate, up = gu.float().chunk(2, dim=1)
    s, g = torch.sigmoid(gate), grad.float()
    return torch.cat([g * up * s * (1 + gate * (1 - s)), g * gate * s], dim=1).to(gu.dtype)


def _to_fp8(w):
    """Weights [E, N, K] as e4m3 with one scale for each expert."""
    top = w.float().abs().amax(dim=(1, 2))
    scale = torch.where(top > 0, top / 448.0, torch.ones_like(top))  # (an expert of zeros)
    return (w.float() / scale[:, None, None]).to(torch.float8_e4m3fn), scale


class MoeLayer:
    """Weights of one layer, 16-bit; `fp8` and `w4` forms are made once by quantize()."""

    def __init__(self, hidden: int, inner: int, experts: int, top_k: int, dtype=torch.bfloat16, seed: int = 0, device="cuda"):
        g = torch.Generator(device=device).manual_seed(seed)

        def randn(*shape, scale):
            return (torch.randn(shape, device=device, generator=g) * scale).to(dtype)

        self.top_k = top_k
        self.norm = torch.ones(hidden, device=device, dtype=torch.float32)
        self.router = randn(experts, hidden, scale=hidden**-0.5)
        self.gate_up = randn(experts, 2 * inner, hidden, scale=hidden**-0.5)
        self.down = randn(experts, hidden, inner, scale=inner**-0.5)

    def quantize(self, group: int = 64) -> None:
        self.gate_up8, self.gate_up_scale = _to_fp8(self.gate_up)
        self.gate_up4, self.down4 = quantize_w4(self.gate_up, group), quantize_w4(self.down, group)

    def forward(self, x, residual, mask=None):
        """(out [T, H], h [T, H], balance loss, what backward takes). mask: False for padding tokens."""
        y, h, rstd, _ = rms_norm(x, self.norm, residual)
        logits = y.float() @ self.router.float().t()
        r = route(logits, self.top_k, mask, balance=True)
        xs = dispatch(y, r)
        gu = grouped_gemm(xs, self.gate_up, r.counts)
        act = _silu_product(gu)
        ys = grouped_gemm(act, self.down, r.counts)
        return combine(ys, r), h, r.loss, (y, h, rstd, logits, r, xs, gu, act, ys)

    def backward(self, saved, grad_out, grad_h=None, grad_loss=None):
        """Gradients by name; "x" is that of x and of residual."""
        y, h, rstd, logits, r, xs, gu, act, ys = saved
        g = {}
        grad_ys, grad_weights = combine_backward(grad_out, ys, r)
        g["down"] = grouped_gemm_wgrad(grad_ys, act, r.counts)
        grad_gu = _silu_product_backward(gu, grouped_gemm_dgrad(grad_ys, self.down, r.counts))
        g["gate_up"] = grouped_gemm_wgrad(grad_gu, xs, r.counts)
        grad_y = dispatch_backward(grouped_gemm_dgrad(grad_gu, self.gate_up, r.counts), r)
        grad_logits = route_backward(logits, r, grad_weights, grad_loss)
        g["router"] = (grad_logits.t() @ y.float()).to(self.router.dtype)
        grad_y = (grad_y.float() + grad_logits @ self.router.float()).to(y.dtype)
        g["x"], g["norm"] = rms_norm_backward(grad_y, h, self.norm, rstd, grad_h)
        return g

    def forward_fp8(self, x, residual):
        """The forward pass with the gate and up products in e4m3: the norm gives their input and its scale. The router reads
        the rounded values, too, so tokens whose experts are close may choose others than in forward; and grouped_gemm_fp8
        takes host sizes, so this pass waits for the counts."""
        y8, h, _, scale = rms_norm(x, self.norm, residual, out_dtype=torch.float8_e4m3fn)
        r = route((y8.float() * scale) @ self.router.float().t(), self.top_k)
        gu = grouped_gemm_fp8(dispatch(y8, r), self.gate_up8, r.counts.tolist(), scale, self.gate_up_scale)
        return combine(grouped_gemm(_silu_product(gu).to(self.down.dtype), self.down, r.counts), r), h

    def decode(self, x, residual):
        """A few tokens, one each of a batch of sequences, on the 4-bit experts. Nothing waits for the GPU."""
        y, h, _, _ = rms_norm(x, self.norm, residual)
        r = route(y.float() @ self.router.float().t(), self.top_k)
        gu = grouped_gemm_w4(dispatch(y, r), self.gate_up4, r.counts)
        return combine(grouped_gemm_w4(_silu_product(gu), self.down4, r.counts), r), h


def _timed(label: str, f):
    f()
    torch.cuda.synchronize()
    t = time.perf_counter()
    for _ in range(10):
        out = f()
    torch.cuda.synchronize()
    print(f"{label:28s} {(time.perf_counter() - t) * 100:8.3f} ms")
    return out


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("tokens", 4096), ("hidden", 2048), ("inner", 1408), ("experts", 32), ("top-k", 4), ("decode", 8)):
        ap.add_argument("--" + name, type=int, default=value)
    a = ap.parse_args()
    layer = MoeLayer(a.hidden, a.inner, a.experts, a.top_k)
    layer.quantize()
    g = torch.Generator(device="cuda").manual_seed(1)
    x, residual, grad = (torch.randn(a.tokens, a.hidden, device="cuda", generator=g).to(torch.bfloat16) for _ in range(3))
    one = torch.full((), 0.01, device="cuda")
    out, _, loss, saved = _timed("forward", lambda: layer.forward(x, residual))
    print(f"{'':28s} balance loss {float(loss):.4f}, rows per expert {int(saved[4].counts.min())} .. {int(saved[4].counts.max())}")
    _timed("backward", lambda: layer.backward(saved, grad, grad, one))
    out8, _ = _timed("forward, fp8 gate and up", lambda: layer.forward_fp8(x, residual))
    print(f"{'':28s} off the 16-bit pass by {float((out8.float() - out.float()).norm() / out.float().norm()):.3f}")
    few, rest = x[:a.decode], residual[:a.decode]
    out4, _ = _timed(f"decode of {a.decode}, 4-bit", lambda: layer.decode(few, rest))
    full, _, _, _ = _timed(f"decode of {a.decode}, 16-bit", lambda: layer.forward(few, rest))
    print(f"{'':28s} off the 16-bit pass by {float((out4.float() - full.float()).norm() / full.float().norm()):.3f}")


if __name__ == "__main__":
    main()
