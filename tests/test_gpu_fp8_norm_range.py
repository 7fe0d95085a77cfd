"""rms_norm_fp8 on rows whose factor is no normal 32-bit number: values below
2^-126 without an eps, values near the largest."""
import pytest
import torch

from oracle import fp8 as O
from test_gpu_fp8 import DT, HALF, TINIEST, check_codes

pytestmark = pytest.mark.gpu

# magnitudes of the rows: bf16 and fp32 share their range, fp16 ends at 2^-24 and 65504
RANGE = {"bf16": [2.0 ** -131, 2.0 ** -126, 2.0 ** -100, 1.0, 2.0 ** 100, 2.0 ** 124],
         "fp32": [2.0 ** -140, 2.0 ** -127, 2.0 ** -100, 1.0, 2.0 ** 100, 2.0 ** 124],
         "fp16": [2.0 ** -22, 2.0 ** -15, 1.0, 2.0 ** 12]}


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T,d", [(6, 64), (7, 130), (12, 2880), (6, 16384), (1203, 1400), (605, 10000)])
@pytest.mark.parametrize("eps", [0.0, 1e-6])
def test_norm_over_the_whole_range(dt, T, d, eps, lib, cuda):
    from moe_stream_b200 import fp8
    g = torch.Generator(device="cuda").manual_seed(T + d)
    size = torch.tensor(RANGE[dt], device="cuda", dtype=torch.float64)[torch.arange(T, device="cuda") % len(RANGE[dt])]
    x = (torch.randn(T, d, generator=g, device="cuda", dtype=torch.float64).clamp(-3.9, 3.9) * size[:, None]).to(DT[dt])
    w = (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(DT[dt])
    assert torch.isfinite(x).all() and (x != 0).any(-1).all()
    q, s, h, y = fp8.rms_norm_fp8(x, w, eps=eps, with_norm=True)
    hx, yx = O.rms_norm(x, w, eps)
    # the factor rounded once, two products rounded: three half steps of 32 bits;
    # below the normal range half a step of 2^-149 a rounding, the first of them
    # and of a value scaled by 2^-64 multiplied by the weight (2 at most) after it
    e = yx.abs() * 3.01 * O.U32 + 2.0 ** -147
    check_codes(q, s, yx, e)
    assert ((y.double() - yx).abs() <= yx.abs() * HALF[dt] + TINIEST[dt] + 1.01 * e).all()


@pytest.mark.parametrize("T,d", [(3, 130), (605, 10000)])
@pytest.mark.parametrize("eps", [1e-6, 1e-60, 1e-100, 1e-200, 1e-300])
def test_rows_of_zeros(T, d, eps, lib, cuda):
    """0 / sqrt(eps) is 0, however small eps is; without one it is NaN."""
    from moe_stream_b200 import fp8
    for dt in DT.values():
        x, w = torch.zeros(T, d, dtype=dt, device="cuda"), torch.ones(d, dtype=dt, device="cuda")
        q, s, h, y = fp8.rms_norm_fp8(x, w, eps=eps, with_norm=True)
        assert (y == 0).all() and (q.float() == 0).all() and (s == 2.0 ** -108).all()
        q, s, h, y = fp8.rms_norm_fp8(x, w, eps=0.0, with_norm=True)
        assert torch.isnan(y).all() and torch.isnan(q.float()).all() and torch.isnan(s).all() and (h == 0).all()
