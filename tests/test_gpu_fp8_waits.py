"""Waits of the fp8 operators that run out, and what follows them.

ms_fp8_selftest_wait enqueues the MoE layer's experts' kernel over a workspace
in which no token is ever routed, so every CTA's wait gives up after its
second: it has to end, report, and leave everything but its own workspace
alone; calls after it are as before, whether the report has been read or not.
No case faults or hangs the GPU: every wait is bounded on the device.
"""
import os
import subprocess
import sys
import textwrap
import threading

import pytest
import torch

from moe_stream_b200 import _lib

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


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
    from moe_stream_b200 import fp8
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


def test_status_gives_up_on_a_stream_that_does_not_finish(lib, cuda):
    """With MS_HOST_WAIT_S=0.2 and a device wait of a second under way,
    ms_fp8_status answers after 0.2 s that the stream did not finish; once it
    has, the report is there, once. In a child process: the limit is read once."""
    code = textwrap.dedent(f"""
        import ctypes, sys, time
        sys.path[:0] = [{ROOT!r}, {os.path.join(ROOT, 'tests')!r}]
        import torch
        from moe_stream_b200 import _lib, fp8
        from test_gpu_fp8_waits import make_layer, tokens
        lib = _lib.load()
        g = torch.Generator(device="cuda").manual_seed(1)
        layer, x = make_layer(g), tokens(g, 20)
        y, ws = torch.empty_like(x), torch.empty(layer._ws[20], dtype=torch.uint8, device="cuda")
        args = layer._pack(x.data_ptr(), 0, y.data_ptr(), ws.data_ptr(), layer._ws[20], 20)
        s = torch.cuda.current_stream().cuda_stream
        st = ctypes.c_int(77)
        layer(x)
        assert lib.ms_fp8_status(0, ctypes.byref(st), s) == 0 and st.value == 0
        t0 = time.monotonic()
        assert lib.ms_fp8_selftest_wait(args, s) == 0
        rc = lib.ms_fp8_status(0, ctypes.byref(st), s)
        host, msg = time.monotonic() - t0, _lib.last_error()
        assert st.value == 0
        torch.cuda.synchronize()
        dev = time.monotonic() - t0
        rc2 = lib.ms_fp8_status(0, ctypes.byref(st), s)
        msg2, st2 = _lib.last_error(), st.value
        rc3 = lib.ms_fp8_status(0, ctypes.byref(st), s)
        print("RESULT", rc, round(host, 3), round(dev, 3), rc2, st2, rc3, st.value, "|", msg, "|", msg2)
    """)
    out = subprocess.run([sys.executable, "-c", code], env=dict(os.environ, MS_HOST_WAIT_S="0.2"), capture_output=True,
                         text=True, timeout=120)
    assert out.returncode == 0, out.stderr[-2000:]
    head, msg, msg2 = [l for l in out.stdout.splitlines() if l.startswith("RESULT")][-1].split("|")
    _, rc, host, dev, rc2, st2, rc3, st3 = head.split()
    assert int(rc) == _lib.MS_E_TIMEOUT and "did not finish" in msg, head + msg
    assert 0.15 <= float(host) < 0.8 and float(dev) >= 0.95, head
    assert int(rc2) == int(st2) == _lib.MS_E_TIMEOUT and "bounded wait ran out" in msg2, head + msg2
    assert int(rc3) == int(st3) == 0, head


def test_status_from_threads_and_streams(lib, cuda):
    """Eight host threads ask at once, each on its own stream, for one report:
    one of them gets it."""
    from moe_stream_b200 import fp8
    g = torch.Generator(device="cuda").manual_seed(2)
    layer = make_layer(g)
    lose(lib, layer, tokens(g, 20), 0xFF)
    streams = [torch.cuda.Stream() for _ in range(8)]
    start, got = threading.Barrier(8), []

    def ask(s):
        start.wait()
        for _ in range(20):
            try:
                fp8.status(0, stream=s)
            except _lib.MoeStreamError as e:
                got.append(e.code)

    threads = [threading.Thread(target=ask, args=(s,)) for s in streams]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert got == [_lib.MS_E_TIMEOUT]


def test_status_is_refused_in_a_capture(lib, cuda):
    """The refusal leaves the capture whole."""
    from moe_stream_b200 import fp8
    g = torch.Generator(device="cuda").manual_seed(3)
    layer, x = make_layer(g), tokens(g, 5)
    want = layer(x)
    fp8.status()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer(x)
        with pytest.raises(_lib.MoeStreamError, match="capture"):
            fp8.status()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want)


def test_status_beside_another_threads_capture():
    """The first question of a process, which sets up the answer's memory, while
    another thread captures: both go through. In a child process, as it has to be
    the first."""
    code = textwrap.dedent(f"""
        import sys, threading
        sys.path[:0] = [{ROOT!r}, {os.path.join(ROOT, 'tests')!r}]
        import torch
        from moe_stream_b200 import fp8
        from test_gpu_fp8_waits import make_layer, tokens
        g = torch.Generator(device="cuda").manual_seed(1)
        layer, x = make_layer(g), tokens(g, 5)
        want, side = layer(x), torch.cuda.Stream()
        torch.cuda.synchronize()
        graph, said = torch.cuda.CUDAGraph(), []
        def ask():
            try:
                fp8.status(0, stream=side)
                said.append("ok")
            except Exception as e:
                said.append(repr(e))
        with torch.cuda.graph(graph, capture_error_mode="global"):
            t = threading.Thread(target=ask)
            t.start(), t.join()
            y = layer(x)
        graph.replay()
        torch.cuda.synchronize()
        print("RESULT", said, torch.equal(y, want))
    """)
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120)
    assert "RESULT ['ok'] True" in out.stdout, out.stdout[-500:] + out.stderr[-1500:]
