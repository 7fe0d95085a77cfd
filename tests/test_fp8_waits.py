"""The fp8 operators' wait self-test on the CPU: what it refuses."""
import pytest


@pytest.mark.parametrize("kw,word", [(dict(T=0), "above 12"), (dict(T=1), "above 12"), (dict(T=12), "above 12"),
                                     (dict(T=65), "T must"), (dict(T=13, nb=16), "workspace is too small"),
                                     (dict(T=13, y=0), "NULL"), (dict(T=13, x=66), "16-byte")])
def test_selftest_refuses(lib, kw, word):
    from moe_stream_b200 import _lib, fp8
    d = dict(x=64, r=64, rb=0, c0=64, c1=64, c2=64, s0=64, s1=64, s2=64, b0=0, b1=0, b2=0, res=0, y=64, ws=64,
             nb=1 << 40, model=0, T=13, d=256, f=128, E=16, k=2, norm=1, device=0)
    d.update(kw)
    assert lib.ms_fp8_selftest_wait(fp8._MOE.pack(*d.values()), None) == _lib.MS_E_INVALID
    assert word in _lib.last_error()
