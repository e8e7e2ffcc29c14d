"""The layer operators without a GPU: the C ABI refuses bad arguments and unsupported shapes before it
touches the device, the torch functions check theirs, the 4-bit storage is what the header says, and
importing the package does not import torch."""
import os
import subprocess
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF16, FP16, E4M3, E5M2, FP32 = 0, 1, 2, 3, 4
INVALID, UNSUPPORTED, WORKSPACE = 2, 1, 4
P = 4096  # an aligned address that is never dereferenced: every call below is refused first


def _refused(pkg, status, want, text):
    msg = pkg.load_library().gg_layer_last_error().decode()
    assert status == want and text in msg, (status, msg)


@pytest.mark.parametrize("change,want,text", [
    (dict(dtype=FP32), INVALID, "dtype"),
    (dict(wdtype=FP16), INVALID, "weight_dtype"),
    (dict(mode=7), INVALID, "scale_mode"),
    (dict(out=E4M3), INVALID, "out_dtype"),
    (dict(mode=1), INVALID, "out_dtype"),
    (dict(mode=2, out=E4M3, scale=None), INVALID, "scale is null"),
    (dict(rows=-1), INVALID, "rows"),
    (dict(hidden=0), INVALID, "hidden"),
    (dict(hidden=100), UNSUPPORTED, "multiple of 8"),
    (dict(hidden=32776), UNSUPPORTED, "at most 32768"),
    (dict(x=None), INVALID, "x is null"),
    (dict(x=P + 8), UNSUPPORTED, "16-byte aligned"),
    (dict(xs=132), UNSUPPORTED, "row strides"),
    (dict(xs=-128), INVALID, "negative"),
    (dict(h=None), INVALID, "h is null"),
    (dict(hs=64), INVALID, "overlap"),
    (dict(y=None), INVALID, "weight and y"),
    (dict(y=P + 8), UNSUPPORTED, "aligned"),
    (dict(mode=1, out=E4M3, ws=None), INVALID, "workspace"),
])
def test_rms_norm_refusals(pkg, change, want, text):
    a = dict(dtype=BF16, wdtype=BF16, out=BF16, mode=0, rows=4, hidden=128, x=P, xs=128, r=P, rs=128, w=P, h=P, hs=128, y=P,
             rstd=P, scale=P, ws=P)
    a.update(change)
    st = pkg.load_library().gg_rms_norm(a["dtype"], a["wdtype"], a["out"], a["mode"], a["rows"], a["hidden"], 1e-6, a["x"], a["xs"],
                                        a["r"], a["rs"], a["w"], a["h"], a["hs"], a["y"], a["rstd"], a["scale"], a["ws"], None)
    _refused(pkg, st, want, text)


@pytest.mark.parametrize("change,want,text", [
    (dict(dtype=E4M3), INVALID, "dtype"),
    (dict(hidden=12), UNSUPPORTED, "multiple of 8"),
    (dict(g=None), INVALID, "grad_y is null"),
    (dict(gx=None), INVALID, "grad_x"),
    (dict(gh=P + 2), UNSUPPORTED, "grad_h"),
    (dict(bytes=16), WORKSPACE, "workspace"),
    (dict(ws=None), WORKSPACE, "workspace"),
])
def test_rms_norm_backward_refusals(pkg, change, want, text):
    lib = pkg.load_library()
    a = dict(dtype=BF16, rows=4, hidden=128, g=P, gh=P, gx=P, ws=P, bytes=lib.gg_rms_norm_backward_workspace(4, 128))
    a.update(change)
    st = lib.gg_rms_norm_backward(a["dtype"], a["dtype"], a["rows"], a["hidden"], a["g"], 128, P, 128, P, P, a["gh"], 128, a["gx"], P,
                                  a["ws"], a["bytes"], None)
    _refused(pkg, st, want, text)


@pytest.mark.parametrize("change,want,text", [
    (dict(dtype=E5M2), INVALID, "dtype"),
    (dict(k=0), INVALID, "top_k"),
    (dict(k=65), INVALID, "top_k"),
    (dict(k=33), UNSUPPORTED, "top_k"),
    (dict(e=1025), UNSUPPORTED, "experts"),
    (dict(t=1 << 29), UNSUPPORTED, "2^31"),
    (dict(t=(1 << 28) + 1, k=2), UNSUPPORTED, "tokens must be at most"),
    (dict(logits=None), INVALID, "logits is null"),
    (dict(logits=P + 2), UNSUPPORTED, "aligned"),
    (dict(stride=-64), INVALID, "negative"),
    (dict(counts=None), INVALID, "counts"),
    (dict(slope=None), INVALID, "loss and slope"),
    (dict(bytes=64), WORKSPACE, "workspace"),
])
def test_route_refusals(pkg, change, want, text):
    lib = pkg.load_library()
    a = dict(dtype=FP32, t=1000, e=64, k=8, logits=P, stride=64, counts=P, slope=P, bytes=lib.gg_route_workspace(1000, 64, 8))
    a.update(change)
    st = lib.gg_route(a["dtype"], a["t"], a["e"], a["k"], 1, a["logits"], a["stride"], None, P, P, a["counts"], P, P, P, P, a["slope"],
                      P, a["bytes"], None)
    _refused(pkg, st, want, text)


def test_route_workspace_sizes(pkg):
    size = pkg.load_library().gg_route_workspace
    assert size(0, 8, 2) == 0 and size(1, 256, 8) == 0 and size(32, 1024, 32) == 0  # one launch
    assert size(4096, 256, 8) >= (4096 // 128) * 256 * 8
    assert size(4096, 256, 64) == 0  # refused by the call


@pytest.mark.parametrize("change,want,text", [
    (dict(es=3), INVALID, "elem_size"),
    (dict(t=-1), INVALID, "tokens"),
    (dict(k=33), UNSUPPORTED, "top_k"),
    (dict(t=1 << 30), UNSUPPORTED, "2^31"),
    (dict(h=100), UNSUPPORTED, "multiple of 16 bytes"),
    (dict(h=1 << 17), UNSUPPORTED, "128 KB"),
    (dict(rows=None), INVALID, "rows"),
    (dict(x=P + 4), UNSUPPORTED, "aligned"),
    (dict(stride=132), UNSUPPORTED, "strides"),
    (dict(stride=-128), INVALID, "negative"),
])
def test_dispatch_refusals(pkg, change, want, text):
    a = dict(es=2, t=8, k=2, h=128, x=P, stride=128, rows=P)
    a.update(change)
    st = pkg.load_library().gg_dispatch(a["es"], a["t"], a["k"], a["h"], 4, a["x"], a["stride"], a["rows"], P, P, None)
    _refused(pkg, st, want, text)


def test_combine_refusals(pkg):
    lib = pkg.load_library()
    _refused(pkg, lib.gg_combine(FP32, 8, 2, 128, P, P, P, P, None), INVALID, "dtype")
    _refused(pkg, lib.gg_combine(BF16, 8, 2, 12, P, P, P, P, None), UNSUPPORTED, "multiple of 16 bytes")
    _refused(pkg, lib.gg_combine(BF16, 8, 2, 128, P, P, None, P, None), INVALID, "weights")
    _refused(pkg, lib.gg_combine(BF16, 8, 2, 128, P + 2, P, P, P, None), UNSUPPORTED, "aligned")
    _refused(pkg, lib.gg_dispatch_backward(BF16, 8, 2, 128, P, None, P, None), INVALID, "rows")
    _refused(pkg, lib.gg_combine_backward(BF16, 8, 2, 128, 4, P, 12, P, P, P, P, P, P, None), UNSUPPORTED, "strides")
    _refused(pkg, lib.gg_combine_backward(BF16, 8, 2, 128, 4, P, 128, P, P, P, P, P, None, None), INVALID, "grad_weights")


@pytest.mark.parametrize("change,want,text", [
    (dict(dtype=E4M3), INVALID, "dtype"),
    (dict(m=-1), INVALID, "total_m"),
    (dict(group=16), UNSUPPORTED, "group"),
    (dict(n=20), UNSUPPORTED, "multiple of 8"),
    (dict(k=160), UNSUPPORTED, "K of group"),
    (dict(n=(1 << 21) + 8), UNSUPPORTED, "at most"),
    (dict(b=8193), UNSUPPORTED, "at most"),
    (dict(m=(1 << 27) + 1), UNSUPPORTED, "rows at most"),
    (dict(lens=None), INVALID, "group_lens"),
    (dict(x=P + 8), UNSUPPORTED, "aligned"),
    (dict(zeros=P + 2), UNSUPPORTED, "aligned"),
])
def test_gemm_w4_refusals(pkg, change, want, text):
    a = dict(dtype=BF16, b=4, m=8, n=64, k=256, group=128, lens=P, x=P, zeros=None)
    a.update(change)
    st = pkg.load_library().gg_gemm_w4(a["dtype"], a["b"], a["m"], a["n"], a["k"], a["group"], a["lens"], None, a["x"], P, P, a["zeros"], P,
                                       None)
    _refused(pkg, st, want, text)


def test_calls_without_work_need_no_gpu(pkg):
    lib = pkg.load_library()
    assert lib.gg_rms_norm(BF16, BF16, BF16, 0, 0, 128, 1e-6, None, 128, None, 0, P, None, 0, None, None, None, None, None) == 0
    assert lib.gg_dispatch(2, 0, 2, 128, 4, None, 128, None, None, None, None) == 0
    assert lib.gg_combine(BF16, 0, 2, 128, None, None, None, None, None) == 0
    assert lib.gg_combine_backward(BF16, 0, 2, 128, 4, None, 128, None, None, None, None, None, None, None) == 0
    assert lib.gg_gemm_w4(BF16, 0, 0, 64, 128, 128, None, None, None, None, None, None, None, None) == 0
    assert lib.gg_gemm_w4(BF16, 2, 0, 64, 128, 128, P, None, None, None, None, None, None, None) == 0


def test_torch_functions_check_their_arguments(pkg):
    x = torch.zeros(4, 64, dtype=torch.bfloat16)
    w = torch.ones(64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="device"):
        pkg.rms_norm(x, w)
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        pkg.rms_norm(x.float(), w)
    with pytest.raises(TypeError, match="logits"):
        pkg.route(torch.zeros(4, 8, dtype=torch.float64), 2)
    with pytest.raises(ValueError, match="device"):
        pkg.route(torch.zeros(4, 8), 2)
    with pytest.raises(ValueError, match="device"):
        pkg.dispatch(x, None)
    q = torch.zeros(2, 24, 128, dtype=torch.uint8)
    s = torch.ones(2, 24, 4, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="uint8"):
        pkg.pack_w4(q.int(), s)
    with pytest.raises(ValueError, match="scales"):
        pkg.pack_w4(q, s.float())
    with pytest.raises(ValueError, match="group must"):
        pkg.pack_w4(q, torch.ones(2, 24, 8, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="zeros"):
        pkg.pack_w4(q, s, s)
    with pytest.raises(ValueError, match="group must"):
        pkg.quantize_w4(torch.zeros(1, 8, 96, dtype=torch.bfloat16), 64)
    with pytest.raises(AttributeError):
        pkg.no_such_operator


@pytest.mark.parametrize("n,k,group", [(16, 128, 128), (24, 160, 32), (40, 320, 64)])
def test_pack_w4_is_the_storage_of_the_header(pkg, n, k, group):
    g = torch.Generator().manual_seed(n * k)
    q = torch.randint(0, 16, (2, n, k), generator=g, dtype=torch.uint8)
    s = torch.rand(2, n, k // group, generator=g).to(torch.float16)
    z = torch.randint(0, 16, (2, n, k // group), generator=g, dtype=torch.uint8)
    w = pkg.pack_w4(q, s, z)
    assert w.packed.shape == (2, -(-n // 16), -(-k // 128), 64, 16) and (w.n, w.k, w.group) == (n, k, group)
    nibble_of = [0, 2, 4, 6, 1, 3, 5, 7]  # k within eight, by nibble
    for b in range(2):
        for row in range(n):
            for col in range(k):
                a, j, inside = col // 8 % 4, col // 32 % 4, col % 8
                piece = w.packed[b, row // 16, col // 128, 16 * a + row % 16]
                nib = nibble_of.index(inside)
                byte = int(piece[4 * j + nib // 2])
                assert (byte >> (4 * (nib % 2))) & 15 == int(q[b, row, col])
            for c in range(k // group):
                assert w.scales[b, row // 16, c, row % 16] == s[b, row, c]
                assert w.zeros[b, row // 16, c, row % 16] == z[b, row, c]


def test_importing_the_package_leaves_torch_alone():
    code = ("import sys, __graft_entry__ as g; p = g.load_package(); assert 'torch' not in sys.modules; p.Routing; "
            "assert 'torch' in sys.modules")
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
