"""The int8 layer's functions on a stream that is not torch's current one, and calls that overlap.

Outputs and workspaces have to be of the memory of the stream that the kernels run on (torch hands a dropped block out
again to the stream it belongs to, while work there may still use it), and two calls at once share nothing.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs an MI355X", allow_module_level=True)

DEV = torch.device("cuda:0")
BF, I8, E4 = torch.bfloat16, torch.int8, torch.float8_e4m3fn


def _inputs(pkg):
    g = torch.Generator(device=DEV).manual_seed(1)

    def randn(*shape):
        return torch.randn(shape, device=DEV, generator=g)

    d = {"x": randn(300, 2048).to(BF), "r": randn(300, 2048).to(BF), "w": randn(2048).to(BF), "wide": randn(700, 2048).to(BF)}
    d["norm"], d["wide_norm"] = pkg.layer_norm(d["x"], d["w"]), pkg.layer_norm(d["wide"], d["w"])
    d["q"] = pkg.quantize_rows(d["x"])
    d["w8"] = pkg.quantize_i8(randn(4, 512, 2048).to(BF))
    d["lens"] = torch.tensor([100, 0, 150, 50], device=DEV)
    d["many8"] = pkg.quantize_i8(randn(70, 64, 2048).to(BF))
    d["many"] = torch.tensor([4] * 70 + [20], device=DEV)[:70]
    d["routing"] = pkg.route(randn(300, 16), 2)
    return d


CALLS = {
    "layer_norm": lambda p, d, s: p.layer_norm(d["x"], d["w"], d["w"], d["r"], stream=s),
    "layer_norm int8": lambda p, d, s: p.layer_norm(d["x"], d["w"], None, d["r"], 1e-5, I8, "row", stream=s),
    "layer_norm tensor scale": lambda p, d, s: p.layer_norm(d["wide"], d["w"], d["w"], out_dtype=E4, stream=s),
    "layer_norm_backward": lambda p, d, s: p.layer_norm_backward(d["r"], d["x"], d["w"], d["norm"].mean, d["norm"].rstd, stream=s),
    "layer_norm_backward, many rows": lambda p, d, s: p.layer_norm_backward(d["wide"], d["wide"], d["w"], d["wide_norm"].mean,
                                                                            d["wide_norm"].rstd, d["wide"], stream=s),
    "rms_norm int8": lambda p, d, s: p.rms_norm(d["x"], d["w"], d["r"], 1e-6, I8, "row", stream=s),
    "silu_product": lambda p, d, s: p.silu_product(d["x"], stream=s),
    "silu_product int8": lambda p, d, s: p.silu_product(d["x"], I8, stream=s),
    "silu_product_backward": lambda p, d, s: p.silu_product_backward(d["r"][:, :1024], d["x"], stream=s),
    "quantize_rows": lambda p, d, s: p.quantize_rows(d["x"], stream=s),
    "dispatch_scaled": lambda p, d, s: p.dispatch_scaled(d["q"].y, d["q"].scale, d["routing"], stream=s),
    "grouped_gemm_i8": lambda p, d, s: p.grouped_gemm_i8(d["q"].y, d["w8"], d["lens"], d["q"].scale, stream=s),
    "grouped_gemm_i8, 16 bits": lambda p, d, s: p.grouped_gemm_i8(d["x"], d["w8"], d["lens"], stream=s),
    "grouped_gemm_i8, host sizes": lambda p, d, s: p.grouped_gemm_i8(d["x"], d["w8"], [100, 0, 150, 50], stream=s),
    "grouped_gemm_i8, many groups": lambda p, d, s: p.grouped_gemm_i8(d["x"][:280], d["many8"], d["many"], stream=s),
}


def _list(out):
    return [out] if isinstance(out, torch.Tensor) else [t for t in out if isinstance(t, torch.Tensor)]


def _bits(t):
    return t.contiguous().reshape(-1).view(torch.uint8)


def _same(a, b):
    return len(a) == len(b) and all(torch.equal(_bits(x), _bits(y)) for x, y in zip(a, b))


def _owner(t):
    """The stream that a tensor's memory belongs to."""
    for seg in torch.cuda.memory_snapshot():
        if seg["address"] <= t.data_ptr() < seg["address"] + seg["total_size"]:
            return seg["stream"]
    raise AssertionError("not in torch's memory")


@pytest.mark.parametrize("name", list(CALLS))
def test_memory_belongs_to_the_stream_of_the_kernels(pkg, monkeypatch, name):
    d = _inputs(pkg)
    want = _list(CALLS[name](pkg, d, None))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    made = []  # owners of all that the call allocates, workspaces too
    for f in ("empty", "empty_like", "tensor"):
        real = getattr(torch, f)

        def spy(*a, real=real, **k):
            t = real(*a, **k)
            made.append(_owner(t) if t.is_cuda else side.cuda_stream)
            return t

        monkeypatch.setattr(torch, f, spy)
    got = _list(CALLS[name](pkg, d, side.cuda_stream))
    monkeypatch.undo()
    side.synchronize()
    assert made and set(made) == {side.cuda_stream}
    assert _same(got, want)
    assert _same(_list(CALLS[name](pkg, d, torch.cuda.current_stream().cuda_stream)), want)


@pytest.mark.parametrize("name", list(CALLS))
def test_calls_at_once(pkg, name):
    """The same call on two streams and on the current one, none ordered after another."""
    d = _inputs(pkg)
    want = _list(CALLS[name](pkg, d, None))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        got += [_list(CALLS[name](pkg, d, s.cuda_stream)) for s in streams] + [_list(CALLS[name](pkg, d, None))]
    torch.cuda.synchronize()
    assert all(_same(g, want) for g in got)


def test_the_functions_follow_torchs_current_stream(pkg):
    d = _inputs(pkg)
    side = torch.cuda.Stream()
    want = pkg.grouped_gemm_i8(d["x"], d["w8"], d["lens"])
    torch.cuda.synchronize()
    a = torch.ones(4096, 4096, device=DEV)
    with torch.cuda.stream(side):
        for _ in range(6):  # some milliseconds of work
            a = a @ a * 2.0**-12
        x = d["x"] * a[0, 0].to(BF)  # the input, after that work
        got = pkg.grouped_gemm_i8(x, d["w8"], d["lens"])
    torch.cuda.synchronize()
    assert torch.equal(got, want)
