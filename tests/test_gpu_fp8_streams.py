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
    """Copies made in a capture belong to its graph, with the calls that read
    them, on its stream and on one that has joined."""
    from moe_stream_b200 import fp8
    side = torch.cuda.Stream()
    g = _gen(2)
    q, s = fp8.quantize_fp8(torch.randn(5, 512, generator=g, device="cuda"))
    w, ws = _weight(g, 640, 512)
    want = fp8.Fp8Linear(w, ws)(q, s)
    moved = _elsewhere(w), _elsewhere(ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        side.wait_stream(torch.cuda.current_stream())
        torch.cuda._sleep(DELAY)
        lin = fp8.Fp8Linear(*moved)
        y, z = lin(q, s), lin(q, s, stream=side)
        torch.cuda.current_stream().wait_stream(side)
    for _ in range(3):
        y.fill_(7.0), z.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(z, want)


def test_tensors_dropped_after_the_call(lib, cuda):
    """Inputs and layers that are dropped as soon as a call on a stream that is
    held up returns: their memory is not used again before it has run."""
    from moe_stream_b200 import fp8
    g = _gen(3)
    T, d, N = 61, 2048, 1536
    side = torch.cuda.Stream()
    x0, r0 = (torch.randn(T, d, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    n0 = (1 + 0.1 * torch.randn(d, generator=g, device="cuda")).to(torch.bfloat16)
    q0, s0 = fp8.quantize_fp8(x0)
    w0, ws0 = _weight(g, N, d)
    router, parts = _moe(g)
    y0 = torch.randn(T, 256, generator=g, device="cuda").to(torch.bfloat16)

    def norm():
        x, n, r = x0.clone(), n0.clone(), r0.clone()
        return lambda **kw: fp8.rms_norm_fp8(x, n, residual=r, **kw)

    def quantize():
        x = x0.clone()
        return lambda **kw: fp8.quantize_fp8(x, **kw)

    def linear():
        layer, q, s = fp8.Fp8Linear(w0.clone(), ws0.clone()), q0.clone(), s0.clone()
        return lambda **kw: (layer(q, s, **kw),)

    def moe():
        layer = fp8.Fp8MoELayer("qwen3", router.clone(), *[tuple(t.clone() for t in p) for p in parts], top_k=2)
        y, r = y0.clone(), y0.clone()
        return lambda **kw: (layer(y, residual=r, **kw),)

    for make in (norm, quantize, linear, moe):
        want = make()()
        torch.cuda.synchronize()
        call = make()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.cuda._sleep(DELAY)
        got = call(stream=side)
        del call
        # whatever was freed is taken and spoilt, on this stream, at once
        spoilt = [torch.full((n,), 0x7F, dtype=torch.uint8, device="cuda")
                  for n in (512, 2048, 4096, 2 * T * d, T * d, N * d, 4 * ws0.numel(), 8 * 384 * 256, 2 * T * 256,
                            2 * router.numel(), 2 * 8 * 384, 4 * 8 * 384, 4 * s0.numel()) for _ in range(6)]
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), make.__name__
        del spoilt, got, want


def test_a_stream_inside_a_capture(lib, cuda):
    """stream= names a stream that has joined the capture: its calls are part of
    the graph, and tensors dropped in between stay what they were."""
    from moe_stream_b200 import fp8
    g = _gen(4)
    T, d, N = 9, 512, 640
    x, r = (torch.randn(T, d, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    n = (1 + 0.1 * torch.randn(d, generator=g, device="cuda")).to(torch.bfloat16)
    bias = torch.randn(N, generator=g, device="cuda").to(torch.bfloat16)      # copied
    first, second = fp8.Fp8Linear(*_weight(g, N, d), bias), fp8.Fp8Linear(*_weight(g, d, N))
    router, parts = _moe(g, d)
    layer = fp8.Fp8MoELayer("qwen3", router, *parts, top_k=2)

    def chain(**kw):
        q, s, h = fp8.rms_norm_fp8(x, n, residual=r, **kw)
        y = first(q, s, **kw)
        q, s = fp8.quantize_fp8(y, **kw)
        y = second(q, s, **kw)
        q, s, h, y = fp8.rms_norm_fp8(y, n, residual=h, with_norm=True, **kw)
        return layer(y, residual=h, **kw)

    want = chain()
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        side.wait_stream(torch.cuda.current_stream())
        a = chain(stream=side)
        b = chain()                       # beside it
        torch.cuda.current_stream().wait_stream(side)
    for _ in range(5):
        a.fill_(7.0), b.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(a, want) and torch.equal(b, want)
