"""Block-scaled fp8 operators on the GPU against their definitions in 64 bits
(oracle/fp8.py, with the error bounds of a 32-bit implementation)."""
import pytest
import torch

from oracle import fp8 as O

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    yield
    from moe_stream_b200 import fp8
    fp8.status()


DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
HALF = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11, "fp32": 2.0 ** -24}
TINIEST = {"bf16": 2.0 ** -134, "fp16": 2.0 ** -25, "fp32": 2.0 ** -150}   # half a subnormal step


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(g, T, d, dt):
    return (torch.randn(T, d, generator=g, device="cuda") * (1 + 15 * (torch.arange(d, device="cuda") % 61 == 3))).to(DT[dt])


def _weight(g, *shape):
    from moe_stream_b200 import fp8
    return fp8.quantize_weight_fp8(torch.randn(*shape, generator=g, device="cuda") * 0.02)


def _poison():
    """Leave freed memory full of NaNs for the next allocations."""
    t = [torch.full((n,), float("nan"), device="cuda") for n in (1 << 10, 1 << 14, 1 << 18, 1 << 22, 1 << 24)]
    del t


def check_codes(q, s, y, e):
    """q, s quantise something within e of y (64 bits): the scale is y's, or
    one that a maximum within e has; the code is within half a step."""
    d = y.shape[-1]
    a, ea = O.group_max(y), O.group_max(e)
    sd = s.double()
    ok = (sd == O.scale_of(a)) | (sd == O.scale_of(a + ea)) | (sd == O.scale_of((a - ea).clamp_min(0.0)))
    assert ok.all(), f"{int((~ok).sum())} scales are off"
    sv = O.spread(sd, d)
    off = (q.double() - y / sv).abs()
    lim = O.e4m3_step((y.abs() + e) / sv) / 2 + e / sv
    assert (off <= lim).all(), f"codes off by up to {float((off / lim).max())} of the limit"


# --------------------------------------------------------------------- norm
@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T,d", [(1, 1), (3, 7), (1, 64), (2, 128), (37, 130), (5, 768), (1, 2048), (33, 2880),
                                 (7, 4097), (2, 8184), (3, 16384)])
@pytest.mark.parametrize("res", [False, True])
def test_norm(dt, T, d, res, lib, cuda):
    from moe_stream_b200 import fp8
    g = _gen(T * 1000 + d)
    x, w = _rows(g, T, d, dt), (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(DT[dt])
    r = _rows(g, T, d, dt) if res else None
    q, s, h, y = fp8.rms_norm_fp8(x, w, eps=1e-6, residual=r, with_norm=True)
    hx, yx = O.rms_norm(x, w, 1e-6, r)
    assert q.dtype is torch.float8_e4m3fn and q.shape == x.shape and s.shape == (T, -(-d // 128))
    assert torch.equal(h, hx)
    # the factor rounded once, two products rounded: three half steps of 32 bits
    e = yx.abs() * 3.01 * O.U32 + 2.0 ** -149
    check_codes(q, s, yx, e)
    assert ((y.double() - yx).abs() <= yx.abs() * HALF[dt] + TINIEST[dt] + 1.01 * e).all()


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T,d", [(1, 1), (4, 100), (37, 768), (9, 2880), (300, 4096), (3, 16384), (2, 5001)])
def test_quantize_is_exact(dt, T, d, lib, cuda):
    from moe_stream_b200 import fp8
    x = _rows(_gen(d), T, d, dt)
    q, s = fp8.quantize_fp8(x)
    qx, sx = O.quantize(x)
    assert torch.equal(s.double(), sx) and torch.equal(q.double(), qx)


def test_quantize_borders(lib, cuda):
    """Values halfway between two codes go to the even one; maxima on the
    border of two scales; zero, tiny, infinite and NaN groups."""
    from moe_stream_b200 import fp8
    x = torch.zeros(10, 256, device="cuda")
    x[0, :128] = torch.arange(128) * 0.5 + 384        # up to 447.5: codes 32 apart
    x[1, 0], x[1, 1] = 448.0, 1.0
    x[2, 0], x[2, 1] = 448.00003, 1.0
    x[3, 5], x[3, 200] = 1e-38, 1e-30
    x[4, 3], x[4, 200] = float("inf"), 1.0
    x[5, 3], x[5, 200] = float("nan"), 1.0
    x[6, 0], x[6, 130] = 3.4e38, -3.4e38
    x[7, :128] = torch.linspace(-2.0 ** -6, 2.0 ** -6, 128)
    x[7, 0] = 448.0                                     # the others are below the normal range
    x[8] = -0.0
    x[9, 127], x[9, 128] = float("-inf"), 2.0
    q, s = fp8.quantize_fp8(x)
    qx, sx = O.quantize(x)
    assert torch.equal(torch.nan_to_num(s.double(), nan=-1.0), torch.nan_to_num(sx, nan=-1.0))
    assert torch.equal(torch.nan_to_num(q.double(), nan=-1000.0), torch.nan_to_num(qx, nan=-1000.0))
    assert torch.isnan(q[4, :128].float()).all() and torch.isfinite(q[4, 128:].float()).all()


def test_norm_rows_that_go_wrong(lib, cuda):
    """A zero row, a row with a NaN, a row with an infinity: the others keep
    their values."""
    from moe_stream_b200 import fp8
    g = _gen(3)
    x, w = _rows(g, 5, 320, "bf16"), torch.ones(320, device="cuda", dtype=torch.bfloat16)
    good, gs, _ = fp8.rms_norm_fp8(x, w)
    x[1] = 0
    x[2, 300] = float("nan")
    x[3, 5] = float("inf")
    q, s, h = fp8.rms_norm_fp8(x, w)
    assert h is x
    for t in (0, 4):
        assert torch.equal(q[t].float(), good[t].float()) and torch.equal(s[t], gs[t])
    assert (q[1].float() == 0).all() and (s[1] == 2.0 ** -108).all()
    assert torch.isnan(q[2].float()).all() and torch.isnan(s[2]).all()
    # an infinity makes the factor 0: itself NaN, its group with it
    assert torch.isnan(s[3, 0]) and (s[3, 1:] == 2.0 ** -108).all() and (q[3, 128:].float() == 0).all()


def test_norm_strides_shapes_and_in_place(lib, cuda):
    from moe_stream_b200 import fp8
    g = _gen(4)
    for d, off in ((256, 8), (256, 3), (200, 0), (250, 1)):
        wide, w = _rows(g, 12, 600, "bf16"), _rows(g, 1, d, "bf16")[0]
        x, r = wide[:, off:off + d], _rows(g, 12, 600, "bf16")[:, 300:300 + d]
        want = fp8.rms_norm_fp8(x.contiguous(), w, residual=r.contiguous(), with_norm=True)
        got = fp8.rms_norm_fp8(x, w, residual=r, with_norm=True)
        for a, b in zip(want, got):
            assert torch.equal(a.float(), b.float())
        # transposed features, three dimensions
        xt = x.t().contiguous().t()
        got = fp8.rms_norm_fp8(xt.reshape(3, 4, d), w, residual=r.reshape(3, 4, d))
        assert got[0].shape == (3, 4, d) and got[1].shape == (3, 4, -(-d // 128))
        assert torch.equal(got[0].float().reshape(12, d), want[0].float())
        for which in (0, 1):
            a, b = x.contiguous().clone(), r.contiguous().clone()
            q, s, h = fp8.rms_norm_fp8(a, w, residual=b, h_out=(a, b)[which])
            assert h is (a, b)[which]
            for p, o in zip((q, s, h), want):
                assert torch.equal(p.float(), o.float())
    assert fp8.rms_norm_fp8(x[0], w)[0].shape == (250,)
    e = fp8.rms_norm_fp8(x[:0], w, residual=r[:0])
    assert e[0].shape == (0, 250) and e[1].shape == (0, 2) and e[2].shape == (0, 250)


@pytest.mark.parametrize("T,d", [(3, 256), (2, 250), (700, 768)])
def test_norm_writes_h_without_a_residual(T, d, lib, cuda):
    """The C entry takes h without a residual: h is x then, in h's own stride."""
    from moe_stream_b200 import fp8
    g = _gen(d)
    x, w = _rows(g, T, d, "bf16"), _rows(g, 1, d, "bf16")[0]
    want = fp8.rms_norm_fp8(x, w)
    wide = torch.full((T, d + 22), 7.0, dtype=torch.bfloat16, device="cuda")
    q, s = torch.empty_like(want[0]), torch.empty_like(want[1])
    dev = x.get_device()
    args = fp8._NORM.pack(x.data_ptr(), 0, w.data_ptr(), wide.data_ptr(), 0, q.data_ptr(), s.data_ptr(),
                          d, 0, d + 22, 0, q.stride(0), 1e-6, T, d, 0, dev)
    assert lib.ms_rms_norm_fp8(args, torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(wide[:, :d], x) and (wide[:, d:] == 7.0).all()
    assert torch.equal(q.view(torch.uint8), want[0].contiguous().view(torch.uint8)) and torch.equal(s, want[1])


def test_norm_offsets_past_32_bits(lib, cuda):
    """More than 2^31 features: rows do not depend on their neighbours."""
    from moe_stream_b200 import fp8
    g = _gen(21)
    T, d = (1 << 20) + 37, 2048
    x = torch.randn(T, d, generator=g, device="cuda", dtype=torch.bfloat16)
    w = _rows(g, 1, d, "bf16")[0]
    for run in (lambda v: fp8.quantize_fp8(v), lambda v: fp8.rms_norm_fp8(v, w, residual=v)):
        got = run(x)
        for at in (0, T // 2, T - 64):
            for a, b in zip(got, run(x[at:at + 64])):
                assert torch.equal(a[at:at + 64].view(torch.uint8), b.view(torch.uint8))
        del got


# ------------------------------------------------------------------- linear
def _codes(g, M, K, pad_with=0x7F):
    """Codes [M, K] in rows padded to 16 bytes with NaN codes, and scales that
    are no powers of two."""
    ld = (K + 15) // 16 * 16
    q = torch.full((M, ld), pad_with, dtype=torch.uint8, device="cuda")
    q[:, :K] = (torch.randn(M, K, generator=g, device="cuda") * 60).to(torch.float8_e4m3fn).view(torch.uint8)
    s = torch.rand(M, -(-K // 128), generator=g, device="cuda") * 0.01 + 0.003
    return q.view(torch.float8_e4m3fn)[:, :K], s


def check_linear(y, xq, xs, wq, ws, bias, dt):
    kb = -(-xq.shape[1] // 128)
    yx, tol = O.product(O.rows_value(xq, xs), O.weight_value(wq, ws), kb)
    if bias is not None:
        yx, tol = yx + bias.double(), tol + O.U32 * (yx.abs() + bias.double().abs())
    off = (y.double() - yx).abs()
    lim = tol + HALF[dt] * (yx.abs() + tol) + TINIEST[dt]
    assert torch.isfinite(off).all() and (off <= lim).all(), f"off by up to {float((off / lim).max())} of the limit"


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 8, 16), (1, 5120, 2048), (2, 130, 127), (3, 64, 128), (16, 2880, 4096),
                                   (17, 129, 129), (31, 500, 320), (33, 513, 1000), (64, 768, 2048), (65, 256, 640),
                                   (100, 2880, 2880), (128, 128, 128), (129, 385, 272), (200, 1024, 96), (256, 256, 256),
                                   (300, 640, 2880), (513, 5120, 400), (1000, 333, 2049),
                                   (333, 5120, 2880), (70, 8200, 1030), (1500, 3000, 1160), (64, 20000, 144)])
def test_linear(M, N, K, dt, lib, cuda):
    from moe_stream_b200 import fp8
    g = _gen(M * 7 + N * 3 + K)
    xq, xs = _codes(g, M, K)
    wq, _ = _codes(g, N, K)
    ws = torch.rand(-(-N // 128), -(-K // 128), generator=g, device="cuda") * 0.01 + 0.003
    bias = torch.randn(N, generator=g, device="cuda").to(torch.bfloat16) if (M + N) % 2 else None
    _poison()
    y = fp8.Fp8Linear(wq, ws, bias)(xq, xs, out_dtype=DT[dt])
    assert y.shape == (M, N) and y.dtype is DT[dt]
    check_linear(y, xq, xs, wq, ws, bias, dt)


def test_linear_large(lib, cuda):
    """The largest shape that is used, in parts; the same rows alone give the
    same bits wherever the same kernel serves both."""
    from moe_stream_b200 import fp8
    g = _gen(11)
    M, N, K = 8200, 5120, 2880
    xq, xs = _codes(g, M, K)
    wq, ws = _weight(g, N, K)
    lin = fp8.Fp8Linear(wq, ws)
    y = lin(xq, xs)
    for m0 in range(0, M, 1024):
        m1 = min(M, m0 + 1024)
        check_linear(y[m0:m1], xq[m0:m1], xs[m0:m1], wq, ws, None, "bf16")
    assert torch.equal(y, lin(xq, xs))


@pytest.mark.parametrize("M,N,K", [(524400, 4104, 128), (524400, 4099, 128), (131300, 136, 16384), (3, 131200, 16400),
                                   (150, 131200, 16400)])
def test_linear_offsets_past_32_bits(M, N, K, lib, cuda):
    """More than 2^31 outputs, by tensor stores and one by one, activations
    and weights: parts at both ends."""
    from moe_stream_b200 import fp8
    g = _gen(M + N)

    def codes(n):
        c = torch.randint(0, 0x60, (n, K), generator=g, device="cuda", dtype=torch.uint8)
        c[:, ::3] |= 0x80
        return c.view(torch.float8_e4m3fn)

    kb = -(-K // 128)
    xq, wq = codes(M), codes(N)
    xs = torch.rand(M, kb, generator=g, device="cuda") + 0.5
    ws = (torch.rand(-(-N // 128), kb, generator=g, device="cuda") + 0.5) * 2.0 ** -12
    y = fp8.Fp8Linear(wq, ws)(xq, xs)
    for m in {0, max(0, M - 130)}:
        for n in {0, (N - 1) // 128 * 128 - 128}:
            check_linear(y[m:m + 130, n:n + 256], xq[m:m + 130], xs[m:m + 130], wq[n:n + 256],
                         ws[n // 128:n // 128 + 2], None, "bf16")


@pytest.mark.parametrize("M", [5, 40, 300])
def test_linear_nan_rows_stay_alone(M, lib, cuda):
    from moe_stream_b200 import fp8
    g = _gen(M)
    N, K = 300, 500
    xq, xs = _codes(g, M, K)
    wq, _ = _codes(g, N, K)
    ws = torch.rand(3, 4, generator=g, device="cuda")
    good = fp8.Fp8Linear(wq, ws)(xq, xs)
    xs2 = xs.clone()
    xs2[1, 2] = float("nan")
    x2 = xq.view(torch.uint8).clone() if xq.is_contiguous() else None
    store = torch.zeros(M, 512, dtype=torch.uint8, device="cuda")
    store[:, :K] = xq.view(torch.uint8) if x2 is None else x2
    store[3, 499] = 0x7F
    y = fp8.Fp8Linear(wq, ws)(store.view(torch.float8_e4m3fn)[:, :K], xs2)
    keep = [m for m in range(M) if m not in (1, 3)]
    assert torch.equal(y[keep], good[keep])
    assert torch.isnan(y[[1, 3]].float()).all()
    wbad = torch.zeros(N, 512, dtype=torch.uint8, device="cuda")
    wbad[:, :K] = wq.view(torch.uint8)
    wbad[17, 250] = 0xFF
    y = fp8.Fp8Linear(wbad.view(torch.float8_e4m3fn)[:, :K], ws)(xq, xs)
    keep = [n for n in range(N) if n != 17]
    assert torch.equal(y[:, keep], good[:, keep]) and torch.isnan(y[:, 17].float()).all()


def test_linear_layouts(lib, cuda):
    """Strided codes and scales, unaligned rows, a transposed weight, out=,
    three dimensions, no rows."""
    from moe_stream_b200 import fp8
    g = _gen(9)
    M, N, K = 24, 260, 384
    xq, xs = _codes(g, M, K)
    wq, _ = _codes(g, N, K)
    ws = torch.rand(3, 3, generator=g, device="cuda")
    want = fp8.Fp8Linear(wq, ws)(xq, xs)
    wide = torch.full((M, 600), 0x7F, dtype=torch.uint8, device="cuda")
    sw = torch.full((M, 9), float("nan"), device="cuda")
    sw[:, 4:7] = xs
    for off in (16, 13):
        wide[:, off:off + K] = xq.view(torch.uint8)
        y = fp8.Fp8Linear(wq, ws)(wide.view(torch.float8_e4m3fn)[:, off:off + K], sw[:, 4:7])
        assert torch.equal(y, want)
        wide.fill_(0x7F)
    wt = wq.view(torch.uint8).t().contiguous().view(torch.float8_e4m3fn).t()
    assert torch.equal(fp8.Fp8Linear(wt, ws)(xq, xs), want)
    lin = fp8.Fp8Linear(wq, ws)
    out = torch.full((2, 12, N), float("nan"), dtype=torch.bfloat16, device="cuda")
    assert lin(xq.reshape(2, 12, K), xs.reshape(2, 12, 3), out=out) is out
    assert torch.equal(out.reshape(M, N), want)
    assert torch.equal(lin(xq[3], xs[3]), lin(xq[3:4], xs[3:4])[0])
    assert lin(xq[:0], xs[:0]).shape == (0, N)
    one = xs[5:6].expand(M, 3)
    assert torch.equal(lin(xq, one), lin(xq, one.contiguous()))


def test_linear_refuses_on_the_gpu(lib, cuda):
    from moe_stream_b200 import fp8
    g = _gen(5)
    xq, xs = _codes(g, 4, 256)
    wq, ws = _weight(g, 128, 256)
    lin = fp8.Fp8Linear(wq, ws)
    for bad, err in ((lambda: lin(xq[:, :255], xs), ValueError), (lambda: lin(xq, xs[:, :1]), ValueError),
                     (lambda: lin(xq, xs[:3]), ValueError), (lambda: lin(xq.float(), xs), TypeError),
                     (lambda: lin(xq, xs.double()), TypeError), (lambda: lin(xq, xs, out_dtype=torch.float64), TypeError),
                     (lambda: lin(xq.cpu(), xs), TypeError),
                     (lambda: lin(xq, xs, out=torch.empty(4, 128, device="cuda")), TypeError),
                     (lambda: lin(xq, xs, out=torch.empty(4, 127, device="cuda", dtype=torch.bfloat16)), ValueError),
                     (lambda: fp8.Fp8Linear(wq, ws[:, :1]), ValueError), (lambda: fp8.Fp8Linear(wq, ws.double()), TypeError),
                     (lambda: fp8.Fp8Linear(wq, ws, bias=torch.zeros(127)), ValueError)):
        with pytest.raises(err):
            bad()


# ---------------------------------------------------------------------- moe
def make_moe(g, model, d, f, E, k, bias=None, norm=True):
    from moe_stream_b200 import fp8
    bias = model == "gptoss" if bias is None else bias
    router = (torch.randn(E, d, generator=g, device="cuda") * 0.05).to(torch.bfloat16)
    rb = (0.1 * torch.randn(E, generator=g, device="cuda")).to(torch.bfloat16) if bias else None
    parts = []
    for n, m in ((f, d), (f, d), (d, f)):
        b = (0.05 * torch.randn(E, n, generator=g, device="cuda")).to(torch.bfloat16) if bias else None
        parts.append((*_weight(g, E, n, m), b))
    layer = fp8.Fp8MoELayer(model, router, *parts, top_k=k, router_bias=rb, norm_topk_prob=norm)
    return layer, router, rb, parts


def _tokens(g, T, d):
    return torch.randn(T, d, generator=g, device="cuda").to(torch.bfloat16)


def check_moe(y, x, router, rb, parts, k, model, norm=True, res=None):
    yx, tol, sure = O.moe_layer(x, router, rb, *parts, k, model, norm, res)
    # tokens whose k-th and next logit are closer than 32 bits tell apart may go either way
    assert sure.double().mean() >= 0.75, "the inputs leave the routing open"
    assert yx.abs().mean() > 8 * tol.mean(), "the bound says nothing about these inputs"
    off = (y.double() - yx).abs()
    assert torch.isfinite(off).all()
    off, tol = off[sure], tol[sure]
    assert (off <= tol).all(), f"off by up to {float((off / tol).max())} of the limit"


@pytest.mark.parametrize("model,T,d,f,E,k", [
    ("qwen3", 1, 256, 128, 8, 2), ("qwen3", 1, 2048, 768, 32, 8), ("qwen3", 3, 320, 192, 16, 4),
    ("qwen3", 8, 512, 768, 60, 8), ("qwen3", 17, 128, 144, 128, 1), ("qwen3", 33, 768, 256, 8, 8),
    ("qwen3", 64, 256, 384, 12, 5), ("gptoss", 1, 2880, 720, 8, 4), ("gptoss", 2, 16, 16, 4, 4),
    ("gptoss", 5, 320, 320, 16, 4), ("gptoss", 64, 272, 400, 32, 4), ("gptoss", 40, 1024, 512, 3, 1),
    ("qwen3", 64, 384, 128, 1, 1), ("qwen3", 2, 256, 256, 256, 32), ("gptoss", 64, 128, 128, 256, 32),
    # many tasks on every SM, tiles cut into ranges by their length
    ("qwen3", 16, 2048, 768, 128, 8), ("gptoss", 5, 2880, 1440, 32, 4), ("qwen3", 61, 1024, 512, 64, 8),
    ("qwen3", 30, 2880, 2880, 4, 2),
    # single tokens: one block, ragged blocks, one expert, many
    ("qwen3", 1, 128, 128, 4, 1), ("gptoss", 1, 272, 144, 16, 4), ("gptoss", 1, 2880, 2880, 4, 4),
    ("qwen3", 1, 400, 656, 256, 32), ("qwen3", 1, 2048, 768, 128, 8), ("gptoss", 1, 4112, 1040, 2, 1)])
def test_moe(model, T, d, f, E, k, lib, cuda):
    g = _gen(T + d + f + E)
    layer, router, rb, parts = make_moe(g, model, d, f, E, k)
    x = _tokens(g, T, d)
    _poison()
    y = layer(x)
    check_moe(y, x, router, rb, parts, k, model)
    r = _tokens(g, T, d)
    check_moe(layer(x, residual=r), x, router, rb, parts, k, model, res=r)
    assert torch.equal(y, layer(x)), "two calls on the same inputs differ"


@pytest.mark.parametrize("T", [1, 6, 40])
def test_moe_offsets_past_32_bits(T, lib, cuda):
    """More than 2^31 codes a matrix; the last experts are the ones chosen."""
    from moe_stream_b200 import fp8
    g = _gen(28)
    d, f, E, k = 2064, 4096, 256, 4
    router = (torch.randn(E, d, generator=g, device="cuda") * 0.05).to(torch.bfloat16)
    rb = torch.zeros(E, device="cuda")
    rb[E - 8:] = 40.0
    parts = []
    for n, m in ((f, d), (f, d), (d, f)):
        c = torch.randint(0, 0x60, (E, n, m), generator=g, device="cuda", dtype=torch.uint8)
        c[:, :, ::3] |= 0x80
        s = (torch.rand(E, -(-n // 128), -(-m // 128), generator=g, device="cuda") + 0.5) * 2.0 ** -10
        parts.append((c.view(torch.float8_e4m3fn), s, None))
    x = _tokens(g, T, d)
    y = fp8.Fp8MoELayer("qwen3", router, *parts, top_k=k, router_bias=rb)(x)
    check_moe(y, x, router, rb, parts, k, "qwen3")


def test_moe_without_renormalisation_and_with_biases(lib, cuda):
    g = _gen(21)
    for bias in (False, True):
        layer, router, rb, parts = make_moe(g, "qwen3", 384, 256, 32, 4, bias=bias, norm=False)
        x = _tokens(g, 6, 384)
        check_moe(layer(x), x, router, rb, parts, 4, "qwen3", norm=False)


def test_moe_clamps(lib, cuda):
    """gpt-oss activations beyond the clamps on both sides."""
    g = _gen(22)
    layer, router, rb, parts = make_moe(g, "gptoss", 256, 256, 4, 2)
    x = (_tokens(g, 9, 256) * 40).to(torch.bfloat16)
    check_moe(layer(x), x, router, rb, parts, 2, "gptoss")


def test_moe_ties_go_to_the_lower_expert(lib, cuda):
    """Equal router rows: the experts chosen are the lowest of them."""
    from moe_stream_b200 import fp8
    g = _gen(23)
    E, d, f, k = 40, 256, 128, 3
    layer, router, rb, parts = make_moe(g, "qwen3", d, f, E, k)
    router = router[:1].expand(E, d).contiguous()
    tied = fp8.Fp8MoELayer("qwen3", router, *parts, top_k=k)
    low = fp8.Fp8MoELayer("qwen3", router[:k].contiguous(), *[(q[:k].contiguous(), s[:k].contiguous()) for q, s, _ in parts],
                          top_k=k)
    x = _tokens(g, 4, d)
    assert torch.equal(tied(x), low(x))


def test_moe_masked_experts_and_nan_tokens(lib, cuda):
    """A router bias of -inf leaves an expert out; a token with a NaN is NaN
    and changes no other token."""
    from moe_stream_b200 import fp8
    g = _gen(24)
    E, d, f, k = 16, 256, 256, 4
    layer, router, _, parts = make_moe(g, "qwen3", d, f, E, k)
    x = _tokens(g, 10, d)
    rb = torch.zeros(E, device="cuda")
    rb[::2] = float("-inf")
    masked = fp8.Fp8MoELayer("qwen3", router, *parts, top_k=k, router_bias=rb)
    keep = fp8.Fp8MoELayer("qwen3", router[1::2].contiguous(),
                           *[(q.view(torch.uint8)[1::2].contiguous().view(q.dtype), s[1::2].contiguous()) for q, s, _ in parts],
                           top_k=k)
    assert torch.equal(masked(x), keep(x))
    want = layer(x)
    x[3, 100] = float("nan")
    x[7] = float("inf")
    y = layer(x)
    others = [t for t in range(10) if t not in (3, 7)]
    assert torch.equal(y[others], want[others])
    assert torch.isnan(y[[3, 7]].float()).all()
    # fewer open experts than top_k: the closed ones weigh nothing
    rb[:] = float("-inf")
    rb[5] = 0.0
    only = fp8.Fp8MoELayer("qwen3", router, *parts, top_k=k, router_bias=rb)(x[:1])
    one = fp8.Fp8MoELayer("qwen3", router[5:6].contiguous(),
                          *[(q.view(torch.uint8)[5:6].contiguous().view(q.dtype), s[5:6].contiguous()) for q, s, _ in parts],
                          top_k=1)(x[:1])
    # another split of the sums: one step of bf16
    assert ((only.double() - one.double()).abs() <= 2.0 ** -7 * one.double().abs()).all()


def test_moe_layouts_and_refusals(lib, cuda):
    from moe_stream_b200 import fp8
    g = _gen(25)
    d, f, E, k = 256, 128, 8, 2
    layer, router, rb, parts = make_moe(g, "qwen3", d, f, E, k)
    x, r = _tokens(g, 6, d), _tokens(g, 6, d)
    want = layer(x, residual=r)
    wide = torch.full((6, 300), float("nan"), dtype=torch.bfloat16, device="cuda")
    wide[:, 5:5 + d] = x
    assert torch.equal(layer(wide[:, 5:5 + d], residual=r.t().contiguous().t()), want)
    assert torch.equal(layer(x.reshape(2, 3, d), residual=r.reshape(2, 3, d)).reshape(6, d), want)
    assert torch.equal(layer(x[2], residual=r[2]), layer(x[2:3], residual=r[2:3])[0])
    a = r.clone()
    assert layer(x, residual=a, out=a) is a and torch.equal(a, want)
    a = x.clone()
    assert torch.equal(layer(a, residual=r, out=a), want)
    assert layer(x[:0]).shape == (0, d)
    for bad, err in ((lambda: layer(_tokens(g, 65, d)), ValueError), (lambda: layer(x.float()), TypeError),
                     (lambda: layer(x[:, :128]), ValueError), (lambda: layer(x, residual=r[:5]), ValueError),
                     (lambda: layer(x, residual=r.float()), TypeError), (lambda: layer(x.cpu()), TypeError),
                     (lambda: layer(x, out=torch.empty(6, d, device="cuda")), TypeError),
                     (lambda: fp8.Fp8MoELayer("qwen3", router, *parts, top_k=9), ValueError),
                     (lambda: fp8.Fp8MoELayer("qwen3", router[:7], *parts, top_k=2), ValueError),
                     (lambda: fp8.Fp8MoELayer("qwen3", router, parts[0], parts[1], parts[0], top_k=2), ValueError),
                     (lambda: fp8.Fp8MoELayer("qwen3", router.float(), *parts, top_k=2), TypeError)):
        with pytest.raises(err):
            bad()


# ----------------------------------------------------------------- together
def make_chain(g, d=320, f=192, E=16, k=4, n=640):
    w1 = (1 + 0.1 * torch.randn(d, generator=g, device="cuda")).to(torch.bfloat16)
    w2 = (1 + 0.1 * torch.randn(d, generator=g, device="cuda")).to(torch.bfloat16)
    return w1, w2, _weight(g, n, d), _weight(g, d, n), make_moe(g, "qwen3", d, f, E, k)


def run_chain(c, x, h):
    """A decoder layer's path with the projections back to back: add + norm,
    a projection, its codes, a projection, add + norm, the MoE layer + add."""
    from moe_stream_b200 import fp8
    w1, w2, a, b, (layer, *_) = c
    q, s, h = fp8.rms_norm_fp8(x, w1, residual=h)
    t = fp8.Fp8Linear(*a)(q, s)
    q, s = fp8.quantize_fp8(t)
    o = fp8.Fp8Linear(*b)(q, s)
    q, s, h2, y = fp8.rms_norm_fp8(o, w2, residual=h, with_norm=True)
    return t, o, h2, y, layer(y, residual=h2), h


def test_chain_against_each_step(lib, cuda):
    """The operators together, each step checked on what the one before gave."""
    from moe_stream_b200 import fp8
    g = _gen(31)
    c = make_chain(g)
    w1, w2, a, b, (layer, router, rb, parts) = c
    for T in (1, 9, 64):
        x, h0 = _tokens(g, T, 320), _tokens(g, T, 320)
        t, o, h2, y, out, h = run_chain(c, x, h0)
        hx, yx = O.rms_norm(x, w1, 1e-6, h0)
        assert torch.equal(h, hx)
        q, s, _ = fp8.rms_norm_fp8(x, w1, residual=h0)
        check_codes(q, s, yx, yx.abs() * 3.01 * O.U32)
        check_linear(t, q, s, *a, None, "bf16")
        q, s = O.quantize(t)
        check_linear(o, q, s, *b, None, "bf16")
        hx, yx = O.rms_norm(o, w2, 1e-6, h)
        assert torch.equal(h2, hx)
        assert ((y.double() - yx).abs() <= yx.abs() * (HALF["bf16"] + 4 * O.U32) + TINIEST["bf16"]).all()
        check_moe(out, y, router, rb, parts, 4, "qwen3", res=h2)


def test_chain_captured_replayed_and_on_other_streams(lib, cuda):
    """The chain in a CUDA graph replayed on new inputs, two graphs of it, the
    chain on two streams at once and with stream= on every call: the same bits
    as alone."""
    from moe_stream_b200 import fp8
    g = _gen(32)
    c = make_chain(g)
    ins = [(_tokens(g, T, 320), _tokens(g, T, 320)) for T in (7, 7, 33, 2)]
    want = [run_chain(c, *i)[:5] for i in ins]
    torch.cuda.synchronize()
    graphs = []
    for n in (0, 2):
        x, h = ins[n][0].clone(), ins[n][1].clone()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = run_chain(c, x, h)[:5]
        graphs.append((gr, x, h, out, n))
    for _ in range(3):
        for gr, x, h, out, n in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for gr, x, h, out, n in graphs:
            for a, b in zip(out, want[n]):
                assert torch.equal(a, b)
    gr, x, h, out, _ = graphs[0]
    x.copy_(ins[1][0]), h.copy_(ins[1][1])
    gr.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want[1]))
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for _ in range(10):
        for n, s in enumerate(streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append((n, run_chain(c, *ins[n])[:5]))
    torch.cuda.synchronize()
    for n, o in got:
        assert all(torch.equal(a, b) for a, b in zip(o, want[n]))
    s = streams[0]
    q, sc, h2 = fp8.rms_norm_fp8(ins[0][0], c[0], residual=ins[0][1], stream=s)
    t = fp8.Fp8Linear(*c[2])(q, sc, stream=s)
    q2, s2 = fp8.quantize_fp8(t, stream=s)
    y = c[4][0](ins[0][0], residual=h2, stream=s)
    s.synchronize()
    assert torch.equal(t, want[0][0])
    qx, sx = O.quantize(t)
    assert torch.equal(q2.double(), qx) and torch.equal(s2.double(), sx)
    assert torch.equal(y, c[4][0](ins[0][0], residual=h2))


def test_layer_on_streams_at_once(lib, cuda):
    """Full layers of one and of many tokens on four streams: whichever SMs a
    call gets, its outputs are those of the call alone."""
    g = _gen(34)
    layer = make_moe(g, "qwen3", 2048, 768, 64, 8)[0]
    xs = [_tokens(g, n, 2048) for n in (1, 1, 20, 64)]
    want = [layer(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    for _ in range(20):
        got = []
        for x, s in zip(xs, streams):
            with torch.cuda.stream(s):
                got.append(layer(x))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_chain_leaves_its_inputs_and_neighbours_alone(lib, cuda):
    """Inputs keep their bits, and rows of a larger buffer next to the output
    keep theirs."""
    from moe_stream_b200 import fp8
    g = _gen(33)
    c = make_chain(g)
    x, h = _tokens(g, 5, 320), _tokens(g, 5, 320)
    x0, h0 = x.clone(), h.clone()
    run_chain(c, x, h)
    assert torch.equal(x, x0) and torch.equal(h, h0)
    lin = fp8.Fp8Linear(*c[2])
    for M in (3, 70, 300):
        q, s = fp8.quantize_fp8(_tokens(g, M, 320))
        buf = torch.full((M + 130, 640), 7.0, dtype=torch.bfloat16, device="cuda")
        lin(q, s, out=buf[1:M + 1])
        assert (buf[0] == 7).all() and (buf[M + 1:] == 7).all() and torch.equal(buf[1:M + 1], lin(q, s))
    layer = c[4][0]
    buf = torch.full((70, 320), 7.0, dtype=torch.bfloat16, device="cuda")
    layer(x, out=buf[4:9])
    assert (buf[:4] == 7).all() and (buf[9:] == 7).all() and torch.equal(buf[4:9], layer(x))
