"""The layer functions on a stream that is not torch's current one.

Memory from torch's allocator belongs to the stream that is current when it is handed out: a dropped tensor's block
goes to the next request on that stream while work queued there still uses it. What a kernel on another stream writes
therefore has to come from that other stream's memory, outputs and workspaces alike.
"""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs an MI355X", allow_module_level=True)

DEV = torch.device("cuda:0")
BF, E4 = torch.bfloat16, torch.float8_e4m3fn
T, E, K, H = 300, 64, 4, 2048  # more than one chunk of the router, so that it needs a workspace


def _inputs(pkg):
    g = torch.Generator(device=DEV).manual_seed(1)

    def randn(*shape):
        return torch.randn(shape, device=DEV, generator=g)

    d = {"x": randn(T, H).to(BF), "r": randn(T, H).to(BF), "w": randn(H).to(BF), "logits": randn(4000, E)}
    d["big"] = pkg.route(d["logits"], K, balance=True)
    d["routing"] = pkg.route(d["logits"][:T].contiguous(), K)
    d["pairs"] = randn(T * K, H).to(BF)
    d["rstd"] = pkg.rms_norm(d["x"], d["w"]).rstd
    d["wide"] = randn(700, 1024).to(BF)  # many rows: the backward pass has a workspace
    d["wide_rstd"] = pkg.rms_norm(d["wide"], d["w"][:1024].contiguous()).rstd
    d["w4"] = pkg.quantize_w4(randn(4, 256, 256).to(BF), 64, True)
    d["few"], d["lens"] = randn(9, 256).to(BF), torch.tensor([4, 0, 3, 2], device=DEV)
    return d


CALLS = {
    "rms_norm": lambda p, d, s: p.rms_norm(d["x"], d["w"], d["r"], stream=s),
    "rms_norm tensor scale": lambda p, d, s: p.rms_norm(d["x"], d["w"], d["r"], out_dtype=E4, stream=s),
    "rms_norm row scale": lambda p, d, s: p.rms_norm(d["x"], d["w"], out_dtype=E4, scale="row", stream=s),
    "rms_norm_backward": lambda p, d, s: p.rms_norm_backward(d["r"], d["x"], d["w"], d["rstd"], stream=s),
    "rms_norm_backward, many rows": lambda p, d, s: p.rms_norm_backward(d["wide"], d["wide"], d["w"][:1024].contiguous(), d["wide_rstd"],
                                                                      stream=s),
    "route": lambda p, d, s: p.route(d["logits"], K, balance=True, stream=s),
    "route_backward": lambda p, d, s: p.route_backward(d["logits"], d["big"], d["big"].weights, d["big"].loss, stream=s),
    "dispatch": lambda p, d, s: p.dispatch(d["x"], d["routing"], stream=s),
    "dispatch_backward": lambda p, d, s: p.dispatch_backward(d["pairs"], d["routing"], stream=s),
    "combine": lambda p, d, s: p.combine(d["pairs"], d["routing"], stream=s),
    "combine_backward": lambda p, d, s: p.combine_backward(d["x"], d["pairs"], d["routing"], stream=s),
    "grouped_gemm_w4": lambda p, d, s: p.grouped_gemm_w4(d["few"], d["w4"], d["lens"], stream=s),
    "grouped_gemm_w4, host sizes": lambda p, d, s: p.grouped_gemm_w4(d["few"], d["w4"], [4, 0, 3, 2], stream=s),
}


def _list(out):
    return [out] if isinstance(out, torch.Tensor) else [t for t in out if isinstance(t, torch.Tensor)]


def _bits(t):
    return t.contiguous().reshape(-1).view(torch.uint8)


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
    inputs = {t.data_ptr() for v in d.values() for t in (_list(v) if isinstance(v, (torch.Tensor, tuple)) else [])}
    assert all(_owner(t) == side.cuda_stream for t in got if t.data_ptr() not in inputs)
    assert len(got) == len(want) and all(torch.equal(_bits(a), _bits(b)) for a, b in zip(got, want))
    # a call on the current stream's own handle is as without one
    assert all(torch.equal(_bits(a), _bits(b)) for a, b in zip(_list(CALLS[name](pkg, d, torch.cuda.current_stream().cuda_stream)), want))


@pytest.mark.parametrize("name", list(CALLS))
def test_work_queued_before_keeps_its_temporaries(pkg, name):
    """Temporaries of the outputs' sizes are dropped while the current stream still has to read them. Then the call,
    with inputs that the other stream is ordered after."""
    d = _inputs(pkg)
    want = _list(CALLS[name](pkg, d, None))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    a = torch.ones(4096, 4096, device=DEV)
    for _ in range(8):  # some milliseconds of work
        a = a @ a * 2.0**-12
    temporaries = [torch.full((_bits(t).numel(),), 77, dtype=torch.uint8, device=DEV) for t in want]
    for _ in range(4):
        a = a @ a * 2.0**-12
    read = [t.clone() for t in temporaries]
    del temporaries
    got = _list(CALLS[name](pkg, d, side.cuda_stream))
    torch.cuda.synchronize()
    assert all(bool((t == 77).all()) for t in read) and bool((a == 1).all())
    assert all(torch.equal(_bits(x), _bits(y)) for x, y in zip(got, want))


def test_outputs_may_be_dropped_while_either_stream_uses_them(pkg):
    """The caller's stream reads an output after an event and drops it; the block is not given out again until then."""
    d = _inputs(pkg)
    want = pkg.rms_norm(d["x"], d["w"], d["r"]).y.clone()
    side, current = torch.cuda.Stream(), torch.cuda.current_stream()
    torch.cuda.synchronize()
    a = torch.ones(4096, 4096, device=DEV)
    y = pkg.rms_norm(d["x"], d["w"], d["r"], stream=side.cuda_stream).y
    current.wait_stream(side)
    for _ in range(8):
        a = a @ a * 2.0**-12
    copy = y.clone()
    place = y.data_ptr()
    del y
    with torch.cuda.stream(side):
        other = torch.zeros_like(want)
        assert other.data_ptr() != place
    torch.cuda.synchronize()
    assert torch.equal(copy, want) and bool((other == 0).all())


def test_the_module_keeps_no_stream(pkg):
    """A refused call on another stream leaves the current stream as it was."""
    d = _inputs(pkg)
    side, current = torch.cuda.Stream(), torch.cuda.current_stream()
    with pytest.raises(pkg.GGError):
        pkg.rms_norm(d["x"][:, :60], d["w"][:60].clone(), stream=side.cuda_stream)
    with pytest.raises(ValueError, match="device"):
        pkg.rms_norm(d["x"].cpu(), d["w"].cpu(), stream=side.cuda_stream)
    assert torch.cuda.current_stream() == current
    assert importlib.import_module(pkg.__name__ + ".moe_layer")._raw_stream(0) == current.cuda_stream
