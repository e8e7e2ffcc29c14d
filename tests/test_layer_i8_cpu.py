"""The operators of an int8 expert layer without a GPU: the C ABI refuses bad arguments and unsupported shapes before it
touches the device, the torch functions check theirs."""
import ctypes
import os
import re

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF16, FP16, E4M3, E5M2, FP32, INT8 = 0, 1, 2, 3, 4, 5
INVALID, UNSUPPORTED, WORKSPACE = 2, 1, 4
P = 4096  # an aligned address that is never dereferenced: every call below is refused first


def _refused(pkg, status, want, text):
    msg = pkg.load_library().gg_layer_last_error().decode()
    assert status == want and text in msg, (status, msg)


@pytest.mark.parametrize("change,want,text", [
    (dict(dtype=FP32), INVALID, "dtype"),
    (dict(wdtype=FP16), INVALID, "weight_dtype"),
    (dict(mode=7), INVALID, "scale_mode"),
    (dict(out=INT8), INVALID, "out_dtype"),
    (dict(mode=1, out=INT8), INVALID, "out_dtype"),
    (dict(mode=3, out=INT8), INVALID, "out_dtype"),
    (dict(mode=2, out=BF16), INVALID, "out_dtype"),
    (dict(mode=2, out=INT8, scale=None), INVALID, "scale is null"),
    (dict(rows=-1), INVALID, "rows"),
    (dict(hidden=100), UNSUPPORTED, "multiple of 8"),
    (dict(hidden=32776), UNSUPPORTED, "at most 32768"),
    (dict(x=None), INVALID, "x is null"),
    (dict(xs=132), UNSUPPORTED, "row strides"),
    (dict(h=None), INVALID, "h is null"),
    (dict(hs=64), INVALID, "overlap"),
    (dict(y=None), INVALID, "weight and y"),
    (dict(b=P + 8), UNSUPPORTED, "aligned"),
    (dict(mode=2, out=INT8, y=P + 4), UNSUPPORTED, "aligned"),
    (dict(mode=1, out=E4M3, ws=None), INVALID, "workspace"),
    (dict(mode=1, out=E4M3, mean=None), INVALID, "mean"),
])
def test_layer_norm_refusals(pkg, change, want, text):
    a = dict(dtype=BF16, wdtype=BF16, out=BF16, mode=0, rows=4, hidden=128, x=P, xs=128, r=P, rs=128, w=P, b=P, h=P, hs=128, y=P,
             mean=P, rstd=P, scale=P, ws=P)
    a.update(change)
    st = pkg.load_library().gg_layer_norm(a["dtype"], a["wdtype"], a["out"], a["mode"], a["rows"], a["hidden"], 1e-5, a["x"], a["xs"],
                                          a["r"], a["rs"], a["w"], a["b"], a["h"], a["hs"], a["y"], a["mean"], a["rstd"], a["scale"],
                                          a["ws"], None)
    _refused(pkg, st, want, text)


@pytest.mark.parametrize("change,want,text", [
    (dict(dtype=INT8), INVALID, "dtype"),
    (dict(hidden=12), UNSUPPORTED, "multiple of 8"),
    (dict(g=None), INVALID, "grad_y is null"),
    (dict(gx=None), INVALID, "grad_x"),
    (dict(mean=None), INVALID, "mean"),
    (dict(gb=None), INVALID, "grad_bias"),
    (dict(gh=P + 2), UNSUPPORTED, "grad_h"),
    (dict(gb=P + 8), UNSUPPORTED, "aligned"),
    (dict(bytes=16), WORKSPACE, "workspace"),
    (dict(ws=None), WORKSPACE, "workspace"),
])
def test_layer_norm_backward_refusals(pkg, change, want, text):
    lib = pkg.load_library()
    a = dict(dtype=BF16, hidden=128, g=P, h=P, w=P, mean=P, rstd=P, gh=P, gx=P, gw=P, gb=P, ws=P,
             bytes=lib.gg_layer_norm_backward_workspace(2000, 128))
    a.update(change)
    st = lib.gg_layer_norm_backward(a["dtype"], a["dtype"], 2000, a["hidden"], a["g"], 128, a["h"], 128, a["w"], a["mean"], a["rstd"],
                                    a["gh"], 128, a["gx"], a["gw"], a["gb"], a["ws"], a["bytes"], None)
    _refused(pkg, st, want, text)


@pytest.mark.parametrize("change,want,text", [
    (dict(dtype=E4M3), INVALID, "dtype"),
    (dict(out=FP16), INVALID, "out_dtype"),
    (dict(rows=-1), INVALID, "rows"),
    (dict(inner=20), UNSUPPORTED, "multiple of 8"),
    (dict(inner=32776), UNSUPPORTED, "at most 32768"),
    (dict(gu=None), INVALID, "gu is null"),
    (dict(stride=132), UNSUPPORTED, "row strides"),
    (dict(y=None), INVALID, "y must be"),
    (dict(y=P + 8), UNSUPPORTED, "aligned"),
    (dict(out=INT8, scale=None), INVALID, "scale"),
    (dict(out=INT8, y=P + 4), UNSUPPORTED, "aligned"),
])
def test_silu_product_refusals(pkg, change, want, text):
    a = dict(dtype=BF16, out=BF16, rows=4, inner=64, gu=P, stride=128, y=P, scale=P)
    a.update(change)
    st = pkg.load_library().gg_silu_product(a["dtype"], a["out"], a["rows"], a["inner"], a["gu"], a["stride"], a["y"], a["scale"], None)
    _refused(pkg, st, want, text)


def test_silu_backward_and_quantize_refusals(pkg):
    lib = pkg.load_library()
    _refused(pkg, lib.gg_silu_product_backward(BF16, 4, 64, None, 64, P, 128, P, None), INVALID, "grad_y is null")
    _refused(pkg, lib.gg_silu_product_backward(BF16, 4, 64, P, 60, P, 128, P, None), UNSUPPORTED, "grad_y")
    _refused(pkg, lib.gg_silu_product_backward(BF16, 4, 64, P, 64, P, 128, None, None), INVALID, "grad_gu")
    _refused(pkg, lib.gg_silu_product_backward(BF16, 4, 64, P, 64, P, 128, P + 8, None), UNSUPPORTED, "grad_gu")
    _refused(pkg, lib.gg_quantize_rows(FP32, 4, 64, P, 64, P, P, None), INVALID, "dtype")
    _refused(pkg, lib.gg_quantize_rows(BF16, 4, 60, P, 64, P, P, None), UNSUPPORTED, "multiple of 8")
    _refused(pkg, lib.gg_quantize_rows(BF16, 4, 64, P, -64, P, P, None), INVALID, "negative")
    _refused(pkg, lib.gg_quantize_rows(BF16, 4, 64, P, 64, P, None, None), INVALID, "scale")
    _refused(pkg, lib.gg_quantize_rows(BF16, 4, 64, P, 64, P + 4, P, None), UNSUPPORTED, "aligned")
    for st in (lib.gg_silu_product(BF16, BF16, 0, 64, None, 0, None, None, None), lib.gg_quantize_rows(BF16, 0, 64, None, 0, None, None, None),
               lib.gg_silu_product_backward(BF16, 0, 64, None, 0, None, 0, None, None)):
        assert st == 0  # no rows: nothing to launch


def test_torch_functions_refuse_host_tensors_and_types(pkg):
    x, w = torch.zeros(4, 64, dtype=torch.bfloat16), torch.ones(64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="device"):
        pkg.layer_norm(x, w)
    with pytest.raises(TypeError, match="bfloat16"):
        pkg.layer_norm(x.float(), w)
    with pytest.raises(TypeError, match="bfloat16"):
        pkg.layer_norm_backward(x, x.float(), w, None, None)
    for f in (pkg.silu_product, pkg.quantize_rows):
        with pytest.raises(ValueError, match="device"):
            f(x)
        with pytest.raises(TypeError, match="bfloat16"):
            f(x.float())


@pytest.mark.parametrize("rows", [600, 1500, 2048, 2049, 4096, 4097, 16640, 1 << 20])
def test_backward_workgroups_fit_the_gpu(pkg, rows):
    """The layer norm's gradient takes no more workgroups than 256 CUs hold at once, by the compiler's report of each
    instance's waves for each of a CU's four SIMDs and its LDS: the numbers are written down, as the workspace's size needs
    them. Every workgroup has rows."""
    path = os.path.join(ROOT, "groupgemm-cktile-optimized_amd", "lib", "resource_usage.txt")
    if not os.path.exists(path):
        pytest.skip("library not built")
    report, name = {}, None
    with open(path, errors="replace") as f:
        for line in f:
            m = re.search(r"Function Name: (\S+)", line)
            if m:  # <type, waves of a row, pieces, with the sums, rows>
                name = re.search(r"center_back_kernelINS0_\w+?ELi(\d+)ELi(\d+)ELb1ELi(\d+)E", m.group(1))
            m = re.search(r"(Occupancy \[waves/SIMD\]|LDS Size \[bytes/block\]): (\d+)", line)
            if m and name:
                report.setdefault(tuple(map(int, name.groups())), {}).setdefault(m.group(1)[:3], []).append(int(m.group(2)))
    assert len(report) >= 11
    for hidden in (8, 512, 520, 1024, 1032, 2048, 2056, 4096, 4104, 6144, 6152, 8192, 8200, 12288, 12296, 16384, 16392, 32768):
        lib = pkg.load_library()
        if lib.gg_layer_norm_backward_workspace(rows, hidden) == 0:
            continue  # few rows
        wpr = 1 if hidden <= 1024 else 4 if hidden <= 8192 else 8
        pieces = min(p for w, p, _ in report if w == wpr and p * 512 * w >= hidden)
        held = {1: 4, 8: 1}.get(wpr) or {2: 3 if rows <= 2048 else 2, 4: 2 if rows <= 4096 else 1}.get(pieces, 3)
        at = report[wpr, pieces, held]
        of_cu = min(min(at["Occ"]) * 4 // max(wpr * held, 4), 160 * 1024 // max(max(at["LDS"]), 1))
        blocks = lib.gg_layer_norm_backward_workspace(rows, hidden) // (8 * hidden)
        assert of_cu >= 1 and (256 if rows >= 1 << 20 else 1) <= blocks <= min(256 * of_cu, -(-rows // held)), (hidden, blocks, at)


# ---- 8-bit integer products ----


@pytest.mark.parametrize("change,want,text", [
    (dict(out_dtype=INT8), INVALID, "out_dtype"),
    (dict(b=-1), INVALID, "group_num"),
    (dict(k=0), INVALID, "k >= 1"),
    (dict(n=60), UNSUPPORTED, "multiple of 8"),
    (dict(k=24), UNSUPPORTED, "K of 16"),
    (dict(k=131072), UNSUPPORTED, "below 131072"),
    (dict(n=2097160), UNSUPPORTED, "2097152"),
    (dict(b=8193), UNSUPPORTED, "8192"),
    (dict(m=(1 << 27) + 1), UNSUPPORTED, "134217728"),
    (dict(m=1 << 27, n=2097152), UNSUPPORTED, "tiles"),
    (dict(lens=None), INVALID, "device pointers"),
    (dict(xs=None), INVALID, "device pointers"),
    (dict(ws=None), INVALID, "device pointers"),
    (dict(x=P + 8), UNSUPPORTED, "aligned"),
    (dict(ws=P + 4), UNSUPPORTED, "aligned"),
    (dict(mem=None), WORKSPACE, "workspace"),
    (dict(mem=P + 8), WORKSPACE, "workspace"),
    (dict(bytes=32), WORKSPACE, "workspace"),
])
def test_gemm_i8_refusals(pkg, change, want, text):
    lib = pkg.load_library()
    a = dict(out_dtype=BF16, b=4, m=16, n=64, k=128, lens=P, x=P, w=P, xs=P, ws=P, out=P, mem=P, bytes=lib.gg_gemm_i8_workspace(4))
    a.update(change)
    st = lib.gg_gemm_i8(a["out_dtype"], a["b"], a["m"], a["n"], a["k"], a["lens"], None, a["x"], a["w"], a["xs"], a["ws"], a["out"],
                        a["mem"], a["bytes"], None)
    _refused(pkg, st, want, text)


def test_int8_is_no_type_of_the_other_products(pkg):
    """The int8 products have an entry point of their own: the plans of the others refuse the type."""
    lib = pkg.load_library()
    assert lib.gg_gemm_i8_workspace(0) == 0 and lib.gg_gemm_i8(BF16, 0, 16, 64, 128, *[None] * 8, 0, None) == 0
    status = ctypes.create_string_buffer(16)  # host memory, which the call writes
    assert lib.gg_call_device_lens(0, INT8, INT8, 2, 16, 64, 128, P, None, P, P, P, P, P, P, 4096, ctypes.addressof(status), None) == INVALID


def test_dispatch_scaled_refusals(pkg):
    lib = pkg.load_library()
    _refused(pkg, lib.gg_dispatch_scaled(1, 4, 2, 64, 8, P, 64, None, P, P, P, P, None), INVALID, "scale")
    _refused(pkg, lib.gg_dispatch_scaled(1, 4, 2, 64, 8, P, 64, P, P, P, P, None, None), INVALID, "scale")
    _refused(pkg, lib.gg_dispatch_scaled(1, 4, 2, 60, 8, P, 64, P, P, P, P, P, None), UNSUPPORTED, "16 bytes")
    _refused(pkg, lib.gg_dispatch_scaled(3, 4, 2, 64, 8, P, 64, P, P, P, P, P, None), INVALID, "elem_size")


def test_quantize_i8_on_the_host(pkg):
    g = torch.Generator().manual_seed(1)
    w = torch.randn(2, 24, 64, generator=g)
    w[1, 5] = 0
    q = pkg.quantize_i8(w)
    s = w.abs().amax(2) / 127
    s[1, 5] = 1.0
    assert q.w.dtype == torch.int8 and torch.equal(q.scales, s) and torch.equal(q.w, (w / s[..., None]).round().to(torch.int8))
    with pytest.raises(ValueError, match="w must be"):
        pkg.quantize_i8(w[0])
    with pytest.raises(ValueError, match="device"):
        pkg.grouped_gemm_i8(torch.zeros(3, 64, dtype=torch.int8), q, [1, 2], torch.ones(3))


def test_quantize_i8_of_what_is_not_finite(pkg):
    """A channel with a NaN or an infinity must not come out as finite numbers; a leaf's scales are no part of its graph."""
    w = torch.ones(1, 4, 16)
    w[0, 1, 3], w[0, 2, 5], w[0, 3] = float("nan"), -float("inf"), 0.0
    q = pkg.quantize_i8(w.requires_grad_())
    s = q.scales[0]
    assert not q.scales.requires_grad and float(s[3]) == 1.0 and bool((q.w[0, 0] == 127).all())
    assert bool(s[1].isnan()) and float(s[2]) == float("inf") and bool((q.w[0, 1:] == 0).all())
    assert bool((q.w[0].float() * s[:, None])[1:3].isnan().all())
