"""Waits of the fp8 operators that run out, and what follows them.

ms_fp8_selftest_wait enqueues the MoE layer's experts' kernel over a workspace
in which no token is ever routed, so every CTA's wait gives up after its
second: it has to end, report, and leave everything but its own workspace
alone; calls after it are as before, whether the report has been read or not.
No case faults or hangs the GPU: every wait is bounded on the device.
"""
import pytest
import torch

pytestmark = pytest.mark.gpu


def make_layer(g, d=256, f=384, E=8, k=2):
    from moe_stream_b200 import fp8
    w = [fp8.quantize_weight_fp8(torch.randn(E, n, m, generator=g, device="cuda") * 0.02)
         for n, m in ((f, d), (f, d), (d, f))]
    return fp8.Fp8MoELayer("qwen3", (torch.randn(E, d, generator=g, device="cuda") * 0.05).to(torch.bfloat16), *w, top_k=k)


def tokens(g, T, d=256):
    return torch.randn(T, d, generator=g, device="cuda").to(torch.bfloat16)


def lose(lib, layer, x, fill):
    """The self-test over a workspace full of `fill` bytes with a margin on
    both sides: (y, margins untouched)."""
    T, nb, margin = x.shape[0], layer._ws[x.shape[0]], 1 << 20
    buf = torch.full((nb + 2 * margin,), fill, dtype=torch.uint8, device="cuda")
    y = torch.full_like(x, 7.0)
    ws = buf.data_ptr() + margin
    args = layer._pack(x.data_ptr(), 0, y.data_ptr(), ws, nb, T)
    assert lib.ms_fp8_selftest_wait(args, torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    return y, bool((buf[:margin] == fill).all() and (buf[margin + nb:] == fill).all())


def expect_timeout():
    from moe_stream_b200 import _lib, fp8
    with pytest.raises(_lib.MoeStreamError) as e:
        fp8.status()
    assert e.value.code == _lib.MS_E_TIMEOUT
    fp8.status()                     # reading cleared it


@pytest.mark.parametrize("T", [13, 17, 40])
@pytest.mark.parametrize("fill", [0x00, 0x7F, 0xFF])
def test_routing_that_never_comes(T, fill, lib, cuda):
    """Whatever the workspace held: the kernel ends and reports, y and what
    lies around the workspace keep their bits."""
    g = torch.Generator(device="cuda").manual_seed(T)
    layer = make_layer(g)
    y, kept = lose(lib, layer, tokens(g, T), fill)
    assert (y == 7.0).all() and kept
    expect_timeout()


def test_calls_after_an_unread_report(lib, cuda):
    """Calls of every kind of kernel after a wait that ran out, before the
    report is read: the same bits as before it."""
    g = torch.Generator(device="cuda").manual_seed(5)
    layer = make_layer(g)
    xs = [tokens(g, T) for T in (1, 5, 20, 64)]
    want = [layer(x) for x in xs]
    lose(lib, layer, xs[2], 0xFF)
    for _ in range(20):
        for x, y in zip(xs, want):
            assert torch.equal(layer(x), y)
    expect_timeout()


def test_a_call_beside_one_that_fails(lib, cuda):
    """Calls on another stream while the self-test's wait is running."""
    g = torch.Generator(device="cuda").manual_seed(6)
    layer = make_layer(g)
    xs = [tokens(g, T) for T in (1, 20, 64)]
    want = [layer(x) for x in xs]
    side = torch.cuda.Stream()
    x, y = tokens(g, 20), torch.empty(20, 256, dtype=torch.bfloat16, device="cuda")
    nb = layer._ws[20]
    ws = torch.empty(nb, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    assert lib.ms_fp8_selftest_wait(layer._pack(x.data_ptr(), 0, y.data_ptr(), ws.data_ptr(), nb, 20), side.cuda_stream) == 0
    got = [layer(x) for x in xs]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    expect_timeout()
