"""Sizes that the fp8 entry points refuse, on the CPU: 32-bit row counts whose
tiles would pass 2^31."""
import pytest

ROWS = (1 << 31) - (1 << 16)


@pytest.mark.parametrize("T", [ROWS + 1, (1 << 31) - 1])
def test_norm_refuses_rows(lib, T):
    from moe_stream_b200 import _lib, fp8
    args = fp8._NORM.pack(64, 0, 64, 0, 0, 64, 64, 128, 0, 0, 0, 128, 1e-6, T, 128, 0, 0)
    assert lib.ms_rms_norm_fp8(args, None) == _lib.MS_E_INVALID and "T must" in _lib.last_error()


@pytest.mark.parametrize("which", ["M", "N", "K"])
@pytest.mark.parametrize("n", [ROWS + 1, (1 << 31) - 1])
def test_linear_refuses_rows(lib, which, n):
    from moe_stream_b200 import _lib, fp8
    d = dict(M=1, N=32, K=128)
    d[which] = n
    ld = (d["K"] + 15) // 16 * 16
    args = fp8._LINEAR.pack(64, 64, 64, 64, 0, 64, ld, -(-d["K"] // 128), ld, d["N"], d["M"], d["N"], d["K"], 0, 0, 0)
    assert lib.ms_linear_fp8(args, None) == _lib.MS_E_INVALID and which in _lib.last_error()
    assert "2147418112" in _lib.last_error()
