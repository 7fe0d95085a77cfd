"""rms_norm_fp8 and quantize_fp8 over many rows, where a CTA takes several rows
and fetches the next one while it works on one: every width of a CTA (32 to 512
threads), three and four chunks a thread, whole and partial last chunks, against
the definition in 64 bits. Row counts leave some CTAs a row more than others."""
import pytest
import torch

from oracle import fp8 as O
from test_gpu_fp8 import DT, HALF, TINIEST, check_codes

pytestmark = pytest.mark.gpu

# features and rows: 16-bit types take up to four chunks of 8 features a thread
WIDE = [(256, 9601), (600, 4801), (1000, 4801), (1400, 2401), (1992, 2401), (2048, 2401), (2880, 1301), (4000, 1301),
        (4096, 1301), (5000, 701), (8184, 701), (10000, 601), (12304, 601), (16384, 601),
        # rows that are no whole chunks, or whose codes are not on 16 bytes
        (250, 9601), (2881, 1301), (776, 4801)]


def _rows(g, T, d, dt):
    scale = 1 + 15 * (torch.arange(d, device="cuda") % 61 == 3)
    return (torch.randn(T, d, generator=g, device="cuda") * scale).to(DT[dt])


def _inputs(T, d, dt):
    g = torch.Generator(device="cuda").manual_seed(T + d)
    return _rows(g, T, d, dt), (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(DT[dt]), _rows(g, T, d, dt)


def _same(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("d,T", WIDE)
@pytest.mark.parametrize("res", [False, True])
def test_norm_of_many_rows(dt, d, T, res, lib, cuda):
    from moe_stream_b200 import fp8
    x, w, r = _inputs(T, d, dt)
    r = r if res else None
    q, s, h, y = fp8.rms_norm_fp8(x, w, eps=1e-6, residual=r, with_norm=True)
    hx, yx = O.rms_norm(x, w, 1e-6, r)
    assert torch.equal(h, hx)
    # the factor rounded once, two products rounded: three half steps of 32 bits
    e = yx.abs() * 3.01 * O.U32 + 2.0 ** -149
    check_codes(q, s, yx, e)
    assert ((y.double() - yx).abs() <= yx.abs() * HALF[dt] + TINIEST[dt] + 1.01 * e).all()


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("d,T", WIDE)
def test_quantize_many_rows_is_exact(dt, d, T, lib, cuda):
    from moe_stream_b200 import fp8
    x = _inputs(T, d, dt)[0]
    q, s = fp8.quantize_fp8(x)
    qx, sx = O.quantize(x)
    assert torch.equal(s.double(), sx) and torch.equal(q.double(), qx)


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("d,T", WIDE)
def test_norm_of_many_rows_in_place(dt, d, T, lib, cuda):
    """h over x and over the residual, while the next row is on its way."""
    from moe_stream_b200 import fp8
    x, w, r = _inputs(T, d, dt)
    want = fp8.rms_norm_fp8(x, w, residual=r, with_norm=True)
    for which in (0, 1):
        a, b = x.clone(), r.clone()
        got = fp8.rms_norm_fp8(a, w, residual=b, h_out=(a, b)[which], with_norm=True)
        assert got[2] is (a, b)[which]
        assert all(_same(p, o) for p, o in zip(got, want))
        assert torch.equal((b, a)[which], (r, x)[which])
    both = x.clone()
    got = fp8.rms_norm_fp8(both, w, residual=both, h_out=both)
    assert all(_same(p, o) for p, o in zip(got, fp8.rms_norm_fp8(x, w, residual=x)))


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("d,T", [(2880, 1301), (10000, 601)])
def test_many_rows_with_strides(dt, d, T, lib, cuda):
    """Rows of wider buffers, on 16-byte boundaries and off them."""
    from moe_stream_b200 import fp8
    x, w, r = _inputs(T, d, dt)
    want = fp8.rms_norm_fp8(x, w, residual=r)
    for off in (16, 3):
        wide = torch.full((2, T, d + 64), float("nan"), device="cuda", dtype=DT[dt])
        wide[0, :, off:off + d], wide[1, :, off:off + d] = x, r
        got = fp8.rms_norm_fp8(wide[0, :, off:off + d], w, residual=wide[1, :, off:off + d])
        assert all(_same(p, o) for p, o in zip(got, want))


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("d,T", [(768, 4801), (2880, 1301), (8192, 701), (16384, 601)])
def test_bad_rows_among_many(dt, d, T, lib, cuda):
    """A NaN or an infinity in one row leaves the rows before and behind it."""
    from moe_stream_b200 import fp8
    x, w, r = _inputs(T, d, dt)
    good = fp8.rms_norm_fp8(x, w, residual=r)
    bad = [0, 5, T // 2, T - 1]
    x[bad[0], 3], x[bad[1], d - 1], x[bad[2], d // 2], x[bad[3], 0] = (float(v) for v in ("nan", "inf", "-inf", "nan"))
    q, s, h = fp8.rms_norm_fp8(x, w, residual=r)
    keep = torch.ones(T, dtype=torch.bool, device="cuda")
    keep[bad] = False
    for a, b in zip((q, s, h), good):
        assert _same(a.float()[keep], b.float()[keep])
    assert torch.isnan(s[[bad[0], bad[3]]]).all()
    assert torch.isnan(s[bad[1], -1]) and (s[bad[1], :-1] == 2.0 ** -108).all()
