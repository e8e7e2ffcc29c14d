"""The int8 products on the few-row kernel, and on the one that the planner takes, where calls overlap, run on streams of
their own or are replayed; and the int8 layer on them. The sums are exact, so every kernel gives the same bits.

tests/test_gpu_i8_streams.py and tests/test_gpu_moe_example_i8.py hold the same of the persistent kernel, which
tests/conftest.py chooses for them.
"""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():
    pytest.skip("needs an MI355X", allow_module_level=True)

DEV = torch.device("cuda:0")
BF, FP, I8 = torch.bfloat16, torch.float16, torch.int8


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


@pytest.fixture(params=["planner", "0", "2", "4"])
def few(request, monkeypatch):
    """The planner's own choice, or an instance of the few-row kernel."""
    monkeypatch.delenv("GG_SMALL")
    if request.param != "planner":
        monkeypatch.setenv("GG_FEW", request.param)
    return request.param


def _persistent(pkg, monkeypatch, f):
    with monkeypatch.context() as m:
        m.delenv("GG_FEW", raising=False)
        m.setenv("GG_SMALL", "0")
        return f()


def _sizes(b, m, seed):
    share = torch.rand(b, generator=torch.Generator().manual_seed(seed)) ** 2
    lens = (share / share.sum() * m).long()
    lens[seed % b] += m - int(lens.sum())
    return lens.to(DEV)


# up to 64 groups the kernel makes its own table, past it a launch before it writes one into the workspace
@pytest.fixture(params=[(4, 30, 520, 1040), (70, 250, 264, 528)], ids=["4 groups", "70 groups"])
def problem(request, pkg):
    """Weights, and three sets of rows and sizes of the same shapes."""
    b, m, n, k = request.param
    g = _gen(b)
    w = pkg.quantize_i8(torch.randn(b, n, k, device=DEV, generator=g).to(BF))
    return w, [(torch.randn(m, k, device=DEV, generator=g).to(BF), _sizes(b, m, 10 + i)) for i in range(3)]


CALLS = {
    "16 bits": lambda p, w, x, lens, s=None: p.grouped_gemm_i8(x, w, lens, stream=s),
    "int8": lambda p, w, x, lens, s=None: p.grouped_gemm_i8((x * 20).to(I8), w, lens, x[:, 0].float().abs().contiguous(), FP, stream=s),
}


@pytest.mark.parametrize("name", list(CALLS))
def test_calls_at_once_on_different_rows_and_sizes(pkg, few, monkeypatch, problem, name):
    w, sets = problem
    want = [_persistent(pkg, monkeypatch, lambda: CALLS[name](pkg, w, *s)) for s in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.current_stream()]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((i, CALLS[name](pkg, w, *sets[i])))
    torch.cuda.synchronize()
    assert all(torch.equal(out, want[i]) for i, out in got)


def test_memory_belongs_to_the_stream_of_the_kernels(pkg, few, monkeypatch, problem):
    w, sets = problem
    want = [_persistent(pkg, monkeypatch, lambda: CALLS["16 bits"](pkg, w, *s)) for s in sets]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    owners = []

    def owner(t):
        return next(seg["stream"] for seg in torch.cuda.memory_snapshot() if seg["address"] <= t.data_ptr() < seg["address"] + seg["total_size"])

    with monkeypatch.context() as m:
        for f in ("empty", "empty_like"):
            def spy(*a, real=getattr(torch, f), **k):
                t = real(*a, **k)
                owners.append(owner(t))
                return t

            m.setattr(torch, f, spy)
        got = [CALLS["16 bits"](pkg, w, *s, side.cuda_stream) for s in sets]
    side.synchronize()
    assert owners and set(owners) == {side.cuda_stream}
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_captured_calls_share_nothing(pkg, few, monkeypatch, problem):
    """Two graphs on two streams at once, eager calls between; every replay reads the rows and sizes of the time."""
    w, sets = problem
    held = [[t.clone() for t in s] for s in sets[:2]]
    for s in held:
        CALLS["16 bits"](pkg, w, *s)
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for g, s in zip(graphs, held):
        with torch.cuda.graph(g):
            outs.append(CALLS["16 bits"](pkg, w, *s))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(3):
        for j, s in enumerate(held):
            for a, b in zip(s, sets[(i + j) % 3]):
                a.copy_(b)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager = CALLS["16 bits"](pkg, w, *sets[2])
        torch.cuda.synchronize()
        want = [_persistent(pkg, monkeypatch, lambda: CALLS["16 bits"](pkg, w, *s)) for s in sets]
        assert torch.equal(eager, want[2])
        for j, out in enumerate(outs):
            assert torch.equal(out, want[(i + j) % 3]), (i, j)


@pytest.mark.parametrize("tokens", [1, 4, 40])
def test_the_int8_layer(pkg, few, monkeypatch, tokens):
    """The layer's pass, eager and captured, gives the bits of the same pass on the persistent kernel."""
    h = 512
    layer = importlib.import_module(pkg.__name__ + ".moe_example").MoeLayer(hidden=h, inner=256, experts=72, top_k=4, norm="layer")
    layer.quantize(64)
    x, residual = (torch.randn(tokens, h, device=DEV, generator=_gen(i)).to(BF) for i in (1, 2))
    want, _ = _persistent(pkg, monkeypatch, lambda: layer.forward_i8(x, residual))
    assert torch.equal(layer.forward_i8(x, residual)[0], want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = layer.forward_i8(x, residual)
    for seed in (5, 6, 7):
        x.copy_(torch.randn(tokens, h, device=DEV, generator=_gen(seed)))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, _persistent(pkg, monkeypatch, lambda: layer.forward_i8(x, residual))[0])
