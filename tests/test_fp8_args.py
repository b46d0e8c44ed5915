"""Arguments that x100_fp8.h refuses, on the host alone: every refusal comes before the device is looked at."""
import ctypes

import pytest

import x100hip as x

P = 1 << 20          # an address that is aligned to everything and never followed
BIG = 1 << 41


def rows(t=x.T_F32, p=P, ld=256, rs=None, cs=None):
    return x.Rows(t, p, ld, rs, cs)


def fp8(p=P, ld=256, scale=P, ls=64):
    return x.Fp8(p, ld, scale, ls)


def refused(f, *a):
    with pytest.raises(x.X100Error) as e:
        f(*a)
    return e.value.code == x.X100_EINVAL


def ok_or_no_device(f, *a):
    """Accepted: runs nothing here (no rows), or ends at the device check."""
    try:
        f(*a)
    except x.X100Error as e:
        return e.code in (x.X100_ENODEV, x.X100_EHIP)
    return True


def test_quant_refusals():
    q = lambda n=8, d=200, r=rows(), o=fp8(): refused(x.quant_fp8, n, d, r, o, None)  # noqa: E731
    assert ok_or_no_device(x.quant_fp8, 0, 200, rows(), fp8(), None)
    assert q(n=-1) and q(n=1 << 24) and q(n=1 << 22, d=5000, r=rows(ld=5000), o=fp8(ld=5008, ls=1 << 22))
    assert q(d=0) and q(d=x.ROWS_MAX_D + 1, r=rows(ld=BIG >> 8), o=fp8(ld=BIG >> 8))
    assert q(r=rows(p=None)) and q(r=rows(ld=199)) and q(r=rows(t=7)) and q(r=rows(p=P + 2)) and q(r=rows(ld=BIG))
    assert q(r=rows(t=x.T_I32)) and q(r=rows(rs=P, cs=P))
    assert q(o=fp8(p=None)) and q(o=fp8(ld=207)) and q(o=fp8(ld=BIG)) and q(o=fp8(scale=None)) and q(o=fp8(scale=P + 2))
    assert q(o=fp8(ls=7)) and q(o=fp8(ls=BIG)) and q(o=None) and q(r=None)


def test_norm_refusals():
    def n(n=8, d=200, r=rows(), dl=None, w=P, eps=1e-6, h=None, ldh=200, o=fp8()):
        return refused(x.add_rmsnorm_fp8, n, d, r, dl, w, eps, h, ldh, o, None)
    assert ok_or_no_device(x.add_rmsnorm_fp8, 0, 200, rows(), rows(), P, 1e-6, 2 * P, 200, fp8(), None)
    assert n(w=None) and n(w=P + 1) and n(eps=-1.0) and n(eps=float("nan")) and n(eps=float("inf"))
    assert n(r=rows(t=x.T_I32, rs=P, cs=P)) and n(dl=rows(), h=None) and n(dl=rows(), h=P + 2, ldh=200)
    assert n(dl=rows(), h=P * 2, ldh=199) and n(dl=rows(ld=100), h=P * 2) and n(dl=rows(), h=P, ldh=200)   # in place: ldh == ld
    assert n(o=fp8(ls=7)) and n(o=fp8(ld=200)) and n(d=0) and n(n=-1)


def test_gemm_refusals():
    def g(M=8, N=300, K=256, a=fp8(), w=fp8(), t=x.T_BF16, c=P, ldc=300):
        return refused(x.gemm_fp8, M, N, K, a, w, t, c, ldc, None)
    for M, N in ((0, 300), (8, 0)):
        assert ok_or_no_device(x.gemm_fp8, M, N, 256, fp8(), fp8(), x.T_F32, P, 300, None)
    assert g(M=-1) and g(N=-1) and g(K=0) and g(K=8) and g(K=24) and g(K=-16) and g(K=(1 << 24) + 16)
    for M, N in ((1 << 18, (1 << 18) + 1), ((1 << 26) + 1, 1), (1, (1 << 26) + 1), (1 << 30, 1 << 20), (2 ** 31 - 1, 2 ** 31 - 1)):
        assert g(M=M, N=N, a=fp8(ls=1 << 31), ldc=1 << 31)
    for bad in (dict(p=None), dict(p=P + 8), dict(ld=240), dict(ld=264), dict(ld=(1 << 24) + 16), dict(scale=None),
                dict(scale=P + 1), dict(ls=BIG)):
        assert g(a=fp8(**bad)) and g(w=fp8(**bad))
    assert g(a=fp8(ls=7)) and g(w=fp8(ls=1)) and g(a=None) and g(w=None)
    assert g(t=x.T_I32) and g(t=5) and g(c=None) and g(c=P + 1) and g(t=x.T_F32, c=P + 2) and g(ldc=299) and g(ldc=BIG)


def test_struct_is_the_header_s():
    assert ctypes.sizeof(x.Fp8) == 32 and x.Fp8.scale.offset == 16
