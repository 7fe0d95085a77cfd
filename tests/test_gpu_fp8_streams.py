"""The fp8 operators on another stream than their tensors' own (stream=)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DELAY = 200_000_000              # cycles that a stream is held up: 0.1 s


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _weight(g, *shape):
    from moe_stream_b200 import fp8
    return fp8.quantize_weight_fp8(torch.randn(*shape, generator=g, device="cuda") * 0.02)


def _elsewhere(t):
    """t's values in another layout: a constructor has to copy them."""
    last = t.view(torch.uint8) if t.dtype is torch.float8_e4m3fn else t
    return last.mT.contiguous().mT.view(t.dtype)


def _spoil(*sizes):
    """Leave freed blocks of these sizes (bytes) full of NaN codes."""
    t = [torch.full((n,), 0x7F, dtype=torch.uint8, device="cuda") for n in sizes for _ in range(3)]
    torch.cuda.synchronize()
    del t


def _moe(g, d=256, f=384, E=8):
    router = (torch.randn(E, d, generator=g, device="cuda") * 0.05).to(torch.bfloat16)
    parts = [(*_weight(g, E, n, m), (0.05 * torch.randn(E, n, generator=g, device="cuda")).to(torch.bfloat16))
             for n, m in ((f, d), (f, d), (d, f))]
    return router, parts


def test_copies_made_by_a_constructor(lib, cuda):
    """A layer that lays out its weights while its stream is held up, called at
    once on another stream: the copies are there."""
    from moe_stream_b200 import fp8
    g = _gen(1)
    M, N, K, E = 5, 640, 512, 8
    q, s = fp8.quantize_fp8(torch.randn(M, K, generator=g, device="cuda"))
    w, ws = _weight(g, N, K)
    b = torch.randn(N, generator=g, device="cuda").to(torch.bfloat16)
    want = fp8.Fp8Linear(w, ws, b)(q, s)
    router, parts = _moe(g)
    x = torch.randn(3, 256, generator=g, device="cuda").to(torch.bfloat16)
    moe_want = fp8.Fp8MoELayer("gptoss", router, *parts, top_k=2, router_bias=torch.zeros(E, device="cuda"))(x)
    moved = (_elsewhere(w), _elsewhere(ws))
    moe_moved = [(_elsewhere(a), _elsewhere(c), e) for a, c, e in parts]
    side = torch.cuda.Stream()
    for _ in range(2):
        _spoil(N * K, 4 * ws.numel(), 4 * N, *(p[0].numel() for p in parts), *(4 * p[1].numel() for p in parts),
               *(4 * p[2].numel() for p in parts))
        torch.cuda._sleep(DELAY)
        y = fp8.Fp8Linear(*moved, b)(q, s, stream=side)
        torch.cuda._sleep(DELAY)
        z = fp8.Fp8MoELayer("gptoss", _elsewhere(router), *moe_moved, top_k=2,
                            router_bias=torch.zeros(E, device="cuda", dtype=torch.bfloat16))(x, stream=side)
        torch.cuda.synchronize()
        assert torch.equal(y, want)
        assert torch.equal(z, moe_want)
        del y, z


def test_constructors_in_a_capture(lib, cuda):
    """Copies made in a capture belong to its graph, with the calls that read them."""
    from moe_stream_b200 import fp8
    g = _gen(2)
    q, s = fp8.quantize_fp8(torch.randn(5, 512, generator=g, device="cuda"))
    w, ws = _weight(g, 640, 512)
    want = fp8.Fp8Linear(w, ws)(q, s)
    moved = _elsewhere(w), _elsewhere(ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = fp8.Fp8Linear(*moved)(q, s)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want)
