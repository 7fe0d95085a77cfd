"""The fp8 operators at the ends of their sizes."""
import pytest
import torch

from oracle import fp8 as O

pytestmark = pytest.mark.gpu


def _codes(g, n, k):
    """Random codes without a NaN, in rows of 16 bytes or a multiple."""
    c = torch.randint(0, 0x60, (n, (k + 15) // 16 * 16), generator=g, device="cuda", dtype=torch.uint8)
    c[:, ::3] |= 0x80
    return c.view(torch.float8_e4m3fn)[:, :k]


@pytest.mark.parametrize("M", [1, 3, 40, 64])
@pytest.mark.parametrize("N,K", [(65535 * 128 + 130, 16), (65536 * 128, 130), (2 * 65536 * 128 + 1, 5)])
def test_linear_of_very_many_outputs(M, N, K, lib, cuda):
    """More than 65535 tiles of outputs for a few rows."""
    from moe_stream_b200 import fp8
    g = torch.Generator(device="cuda").manual_seed(M + K)
    kb = -(-K // 128)
    x, w = _codes(g, M, K), _codes(g, N, K)
    xs = torch.rand(M, kb, generator=g, device="cuda") + 0.5
    ws = (torch.rand(-(-N // 128), kb, generator=g, device="cuda") + 0.5) * 2.0 ** -12
    y = fp8.Fp8Linear(w, ws)(x, xs)
    assert y.shape == (M, N)
    for n in (0, 65535 * 128 - 128, 65535 * 128, (N - 1) // 128 * 128):
        part = slice(n, min(N, n + 128))
        want, tol = O.product(O.rows_value(x, xs), O.weight_value(w[part], ws[n // 128:n // 128 + 1]), kb)
        lim = tol + 2.0 ** -8 * (want.abs() + tol)
        assert ((y[:, part].double() - want).abs() <= lim).all(), n


def test_row_counts_beyond_the_limit(lib, cuda):
    """2^31 rows and those just below are refused, by expanded tensors that
    hold one row."""
    from moe_stream_b200 import fp8
    one = torch.ones(1, 1, dtype=torch.bfloat16, device="cuda")
    q, s = fp8.quantize_fp8(one)
    w = torch.zeros(16, 1, device="cuda").to(torch.float8_e4m3fn)
    lin = fp8.Fp8Linear(w, torch.ones(1, 1, device="cuda"))
    for T in (1 << 31, (1 << 31) - 1, (1 << 31) - (1 << 16) + 1):
        for bad in (lambda: fp8.quantize_fp8(one.expand(T, 1)), lambda: fp8.rms_norm_fp8(one.expand(T, 1), one[0]),
                    lambda: lin(q.expand(T, 1), s.expand(T, 1)),
                    lambda: fp8.Fp8Linear(w[:1].expand(T, 1), torch.ones(1, 1, device="cuda").expand(-(-T // 128), 1))):
            with pytest.raises(ValueError, match="rows"):
                bad()
    q2, s2 = fp8.quantize_fp8(one)
    assert torch.equal(q2.double(), q.double()) and torch.equal(s2, s)


@pytest.mark.parametrize("M", [2, 15, 16, 17, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257])
@pytest.mark.parametrize("N,K", [(256, 256), (257, 1025), (640, 1152)])
def test_linear_around_the_tiles(M, N, K, lib, cuda):
    """Row counts on both sides of every tile of the kernels and of the choice
    between them."""
    from moe_stream_b200 import fp8
    from test_gpu_fp8 import check_linear
    g = torch.Generator(device="cuda").manual_seed(M + N)
    kb = -(-K // 128)
    x, w = _codes(g, M, K), _codes(g, N, K)
    xs = torch.rand(M, kb, generator=g, device="cuda") + 0.5
    ws = (torch.rand(-(-N // 128), kb, generator=g, device="cuda") + 0.5) * 2.0 ** -12
    check_linear(fp8.Fp8Linear(w, ws)(x, xs, out_dtype=torch.float32), x, xs, w, ws, None, "fp32")


@pytest.mark.parametrize("model", ["qwen3", "gptoss"])
@pytest.mark.parametrize("T", [2, 3, 4, 5, 11, 12, 13, 15, 16, 17, 31, 32, 33, 63, 64])
def test_moe_around_the_tiles(model, T, lib, cuda):
    """Token counts on both sides of every choice: routing by each CTA or
    shared out, tokens of a route CTA, rows of an expert's tile."""
    from test_gpu_fp8 import check_moe, make_moe
    g = torch.Generator(device="cuda").manual_seed(T)
    layer, router, rb, parts = make_moe(g, model, 320, 272, 24, 4)
    x = torch.randn(T, 320, generator=g, device="cuda").to(torch.bfloat16)
    y = layer(x)
    check_moe(y, x, router, rb, parts, 4, model)
    for _ in range(3):
        assert torch.equal(layer(x), y)
