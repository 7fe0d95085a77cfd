"""Block-scaled fp8 operators on the CPU: the 64-bit oracle against known
values, and everything that is refused before a GPU is touched."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import fp8 as O


# ------------------------------------------------------------------ oracle
def test_oracle_e4m3_is_torchs_conversion():
    g = torch.Generator().manual_seed(0)
    v = torch.cat([torch.randn(4096, generator=g) * 100, torch.randn(4096, generator=g) * 2e-3,
                   torch.tensor([0.0, 448.0, 460.0, 2.0 ** -9, 2.0 ** -10, 3 * 2.0 ** -10, 17.0, 19.0, -17.0])])
    v = v.clamp(-464.0, 464.0)
    assert torch.equal(O.e4m3(v.double()), v.to(torch.float8_e4m3fn).double())


def test_oracle_scale_is_the_smallest_power_of_two():
    a = torch.tensor([448.0, 448.1, 447.9, 1.75, 1.7500001, 1.0, 0.0, 1e-38, 3e38, float("inf"), float("nan")])
    s = O.scale_of(a)
    assert s[:6].tolist() == [1.0, 2.0, 1.0, 2.0 ** -8, 2.0 ** -7, 2.0 ** -8]
    assert s[6] == s[7] == 2.0 ** -108 and torch.isnan(s[9:]).all()
    fin = a[:9].double().clamp_min(O.TINY)
    assert (fin <= 448.0 * s[:9]).all() and (fin > 224.0 * s[:9]).all()


def test_oracle_bounds_hold_for_a_32_bit_computation():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(5, 320, generator=g)
    q, s = O.quantize(x)
    w = torch.randn(200, 320, generator=g).to(torch.float8_e4m3fn)
    ws = torch.rand(2, 3, generator=g)
    xv, wv = O.rows_value(q, s), O.weight_value(w, ws)
    y, tol = O.product(xv, wv, 3)
    assert ((xv.float() @ wv.float().T).double() - y).abs().le(tol).all()
    # a missing feature is seen
    xv[:, 7] = 0.0
    assert ((xv @ wv.T) - y).abs().gt(tol).any()


def test_weight_quantiser():
    from moe_stream_b200 import fp8
    g = torch.Generator().manual_seed(2)
    w = torch.randn(3, 200, 300, generator=g) * 0.02
    w[0, :128, :128] = 0.0
    q, s = fp8.quantize_weight_fp8(w)
    assert q.dtype is torch.float8_e4m3fn and s.shape == (3, 2, 3) and s.dtype is torch.float32
    # half a step of e4m3 (2^-4 of the value, 2^-10 of the scale below its
    # normal range) and of the 32-bit quotient and scale
    sv = O.spread(O.spread(s.double(), 200, -2), 300)
    assert ((q.double() * sv - w.double()).abs() <= w.double().abs() * (2.0 ** -4 + 4 * O.U32) + sv * 2.0 ** -10).all()


# ---------------------------------------------------------------- refusals
def _norm(lib, **kw):
    from moe_stream_b200 import fp8
    d = dict(x=64, res=0, w=64, h=0, y=0, q=64, s=64, xs=128, rs=128, hs=128, ys=128, qs=128, eps=1e-6, T=1, d=128,
             dtype=0, device=0)
    d.update(kw)
    return lib.ms_rms_norm_fp8(fp8._NORM.pack(*d.values()), None)


@pytest.mark.parametrize("kw,word", [
    (dict(x=0), "NULL"), (dict(q=0), "NULL"), (dict(s=0), "NULL"), (dict(T=-1), "T must"), (dict(d=0), "d must"),
    (dict(d=16385, qs=16400), "d must"), (dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"),
    (dict(res=64), "needs h"), (dict(w=0, res=64, h=64), "need a weight"), (dict(w=0, y=64), "need a weight"),
    (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(qs=127), "q_stride"),
    (dict(res=64, h=64, hs=127), "h_stride"), (dict(y=64, ys=5), "h_stride or y_stride")])
def test_norm_refuses(lib, kw, word):
    from moe_stream_b200 import _lib
    assert _norm(lib, **kw) == _lib.MS_E_INVALID
    assert word in _lib.last_error()


def _linear(lib, **kw):
    from moe_stream_b200 import fp8
    d = dict(x=64, xs=64, w=64, ws=64, b=0, y=64, ldx=128, lds=1, ldw=128, ldy=32, M=1, N=32, K=128, out=0, device=0,
             pad=0)
    d.update(kw)
    return lib.ms_linear_fp8(fp8._LINEAR.pack(*d.values()), None)


@pytest.mark.parametrize("kw,word", [
    (dict(x=0), "NULL"), (dict(xs=0), "NULL"), (dict(w=0), "NULL"), (dict(ws=0), "NULL"), (dict(y=0), "NULL"),
    (dict(M=-1), "M must"), (dict(N=0), "N and K"), (dict(K=0), "N and K"), (dict(out=7), "out_dtype"),
    (dict(x=72), "16-byte"), (dict(w=65), "16-byte"), (dict(ldx=136), "16-byte"), (dict(ldw=130), "16-byte"),
    (dict(ldx=112), "stride"), (dict(ldw=112), "stride"), (dict(ldy=31), "stride"), (dict(K=129, ldx=144, ldw=144), "stride")])
def test_linear_refuses(lib, kw, word):
    from moe_stream_b200 import _lib
    assert _linear(lib, **kw) == _lib.MS_E_INVALID
    assert word in _lib.last_error()


def _moe(lib, call=True, **kw):
    from moe_stream_b200 import fp8
    d = dict(x=64, r=64, rb=0, c0=64, c1=64, c2=64, s0=64, s1=64, s2=64, b0=0, b1=0, b2=0, res=0, y=64, ws=64,
             nb=1 << 40, model=0, T=1, d=256, f=128, E=8, k=2, norm=1, device=0)
    d.update(kw)
    packed = fp8._MOE.pack(*d.values())
    if call:
        return lib.ms_moe_fp8_layer(packed, None)
    n = ctypes.c_size_t()
    rc = lib.ms_moe_fp8_workspace(packed, ctypes.byref(n))
    return rc, n.value


@pytest.mark.parametrize("kw,word", [
    (dict(model=2), "model"), (dict(T=-1), "T must"), (dict(T=65), "T must"), (dict(E=0), "n_experts"),
    (dict(E=257), "n_experts"), (dict(k=0), "top_k"), (dict(k=9), "top_k"), (dict(E=64, k=33), "top_k"),
    (dict(d=264), "multiples of 16"), (dict(f=0), "multiples of 16"), (dict(f=16400), "multiples of 16")])
def test_moe_refuses_sizes(lib, kw, word):
    from moe_stream_b200 import _lib
    for call in (True, False):
        rc = _moe(lib, call, **kw)
        assert (rc if call else rc[0]) == _lib.MS_E_INVALID
        assert word in _lib.last_error()


@pytest.mark.parametrize("kw,word", [
    (dict(x=0), "NULL"), (dict(r=0), "NULL"), (dict(y=0), "NULL"), (dict(ws=0), "NULL"), (dict(c1=0), "NULL"),
    (dict(s2=0), "NULL"), (dict(c2=72), "16-byte"), (dict(x=66), "16-byte"), (dict(res=8), "16-byte"),
    (dict(nb=16), "workspace is too small")])
def test_moe_refuses_buffers(lib, kw, word):
    from moe_stream_b200 import _lib
    assert _moe(lib, **kw) == _lib.MS_E_INVALID
    assert word in _lib.last_error()


def test_no_rows_is_no_work(lib):
    """Calls over no rows return before they look at a device or a buffer."""
    assert _norm(lib, T=0, x=0) == 0 and _linear(lib, M=0, x=0) == 0 and _moe(lib, T=0, x=0) == 0


def test_workspace_grows_with_the_call(lib):
    sizes = [_moe(lib, False, T=T)[1] for T in (1, 2, 7, 64)]
    assert sizes == sorted(sizes) and sizes[0] > 0


def test_cpu_tensors_are_refused(lib):
    from moe_stream_b200 import fp8
    x, w = torch.zeros(2, 128, dtype=torch.bfloat16), torch.zeros(128, dtype=torch.bfloat16)
    with pytest.raises(TypeError, match="CUDA"):
        fp8.rms_norm_fp8(x, w)
    with pytest.raises(TypeError, match="CUDA"):
        fp8.quantize_fp8(x)
    q, s = fp8.quantize_weight_fp8(torch.zeros(128, 128))
    with pytest.raises(TypeError, match="CUDA"):
        fp8.Fp8Linear(q, s)
    with pytest.raises(TypeError, match="CUDA"):
        fp8.Fp8MoELayer("qwen3", torch.zeros(8, 128, dtype=torch.bfloat16), (q, s), (q, s), (q, s), 2)
    with pytest.raises(ValueError, match="model"):
        fp8.Fp8MoELayer("other", torch.zeros(8, 128, dtype=torch.bfloat16), (q, s), (q, s), (q, s), 2)
    with pytest.raises(TypeError, match="bfloat16"):
        fp8.quantize_fp8(torch.zeros(2, 128, dtype=torch.float64))
    with pytest.raises(TypeError, match="weight"):
        fp8.rms_norm_fp8(x, None)


def test_argument_blocks_have_the_headers_sizes():
    """The packed blocks are laid out as the C structs: 8-byte members first,
    no padding between."""
    from moe_stream_b200 import fp8
    assert (fp8._NORM.size, fp8._LINEAR.size, fp8._MOE.size) == (120, 104, 160)
    assert np.dtype("P").itemsize == 8
