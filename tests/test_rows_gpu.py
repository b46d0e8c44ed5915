"""x100_add_rmsnorm_i8_hip / x100_quant_i8_hip against the definition: codes bit for bit (they do not
depend on the order of a sum), scales within the sum's fp32 error."""
import numpy as np
import pytest
import torch

import paged_ref as ref
import x100hip as x

pytestmark = pytest.mark.gpu

TT = {ref.F32: torch.float32, ref.F16: torch.float16, ref.BF16: torch.bfloat16, ref.I32: torch.int32}
EPS = 1e-6


def stream():
    return torch.cuda.current_stream().cuda_stream


def make(g, n, d, t, pad=0, off=0):
    """Rows of a type: (device buffer, Rows, fp32 values, what keeps scales alive)."""
    if t == ref.I32:
        a = torch.from_numpy(g.integers(-200000, 200000, (n, d + pad)).astype(np.int32))
        rs = torch.from_numpy((g.random(n) * 1e-2 + 1e-4).astype(np.float32))
        cs = torch.from_numpy((g.random(d) * 1e-2 + 1e-4).astype(np.float32))
        vals = (a[:, :d].float() * rs[:, None]) * cs
    else:
        a = torch.from_numpy((g.standard_normal((n, d + pad)) * 3).astype(np.float32)).to(TT[t])
        rs = cs = None
        vals = a[:, :d].float()
    buf = torch.zeros(off + a.numel(), dtype=a.dtype, device="cuda")
    buf[off:] = a.reshape(-1).cuda()
    keep = [buf] + [s.cuda() for s in (rs, cs) if s is not None]
    r = x.Rows(t, buf.data_ptr() + off * buf.element_size(), d + pad, *([k.data_ptr() for k in keep[1:]] or [None, None]))
    return buf, r, vals.numpy(), keep


def check(q, scale, t, factor, n, d):
    """codes of t (fp32) exactly; scale = amax * factor / 127 (factor float64 [n])."""
    want, amax = ref.codes_f32(t)
    q, scale = q.cpu().numpy(), scale.cpu().numpy().astype(np.float64)
    assert np.array_equal(q, want)
    s = amax.astype(np.float64) * factor / 127
    # the sum of d squares, the mean, the root, the quotient and two products in fp32: at most d + 8
    # roundings, the root halves those of the sum
    bound = np.abs(s) * (d / 2 + 8) * 2.0 ** -24
    nan = np.isnan(s)
    assert np.array_equal(nan, np.isnan(scale))
    assert (np.abs(scale - s)[~nan] <= bound[~nan]).all()


SIZES = [(1, 1), (3, 7), (2, 8), (5, 64), (4, 511), (4, 512), (3, 513), (7, 520), (3, 1000), (2, 2048), (2, 2049),
         (3, 2056), (2, 4096), (1, 4104), (2, 5000), (1, 8192), (1, 16383), (2, 16384), (300, 24)]


@pytest.mark.parametrize("t", [ref.F32, ref.F16, ref.BF16, ref.I32])
@pytest.mark.parametrize("n,d", SIZES)
def test_quant(dev, n, d, t):
    g = np.random.default_rng(n * 100003 + d)
    for pad, off in ((0, 0), (8, 0), (3, 1)):
        buf, r, vals, keep = make(g, n, d, t, pad, off)
        q = torch.full((n * d + 16,), 99, dtype=torch.int8, device=dev)
        sc = torch.full((n + 4,), 7.0, device=dev)
        x.quant_i8(n, d, r, q.data_ptr(), sc.data_ptr(), stream())
        torch.cuda.synchronize()
        check(q[:n * d].view(n, d), sc[:n], vals, np.ones(n), n, d)
        assert (q[n * d:] == 99).all() and (sc[n:] == 7).all()


@pytest.mark.parametrize("xt", [ref.F32, ref.F16, ref.BF16])
@pytest.mark.parametrize("dt", [None, ref.F32, ref.F16, ref.BF16, ref.I32])
@pytest.mark.parametrize("n,d", [(1, 1), (3, 63), (5, 512), (3, 1030), (4, 2048), (2, 4096), (3, 4099), (2, 8200), (1, 16384)])
def test_add_rmsnorm(dev, n, d, xt, dt):
    g = np.random.default_rng(n * 7919 + d)
    w = (1 + 0.3 * g.standard_normal(d)).astype(np.float32)
    dw = torch.from_numpy(w).cuda()
    for pad, off, inplace in ((0, 0, False), (0, 0, True), (16, 8, False), (5, 3, True)):
        buf, r, vals, keep = make(g, n, d, xt, pad, off)
        q = torch.full((n, d), 99, dtype=torch.int8, device=dev)
        sc = torch.empty(n, device=dev)
        before = buf.clone()
        if dt is None:
            x.add_rmsnorm_i8(n, d, r, None, dw.data_ptr(), EPS, None, 0, q.data_ptr(), sc.data_ptr(), stream())
            h = vals
            torch.cuda.synchronize()
            assert torch.equal(before, buf)
        else:
            dbuf, dr, dvals, dkeep = make(g, n, d, dt, pad, off)
            hb = buf if inplace else torch.zeros_like(buf)
            x.add_rmsnorm_i8(n, d, r, dr, dw.data_ptr(), EPS, hb.data_ptr() + off * hb.element_size(), d + pad,
                             q.data_ptr(), sc.data_ptr(), stream())
            torch.cuda.synchronize()
            got = hb[off:].view(n, d + pad)
            h = torch.from_numpy(vals + dvals).to(TT[xt])
            assert torch.equal(got[:, :d].cpu(), h)
            if pad:   # what lies between the rows is not touched
                want = before[off:].view(n, d + pad)[:, d:] if inplace else torch.zeros(n, pad, dtype=hb.dtype, device=dev)
                assert torch.equal(got[:, d:], want)
            h = h.float().numpy()
        r64 = 1 / np.sqrt((h.astype(np.float64) ** 2).mean(1) + EPS)
        check(q, sc, h * w, r64, n, d)


@pytest.mark.parametrize("d", [8, 100, 2048, 8192])
def test_rows_of_zeros_infinities_nan(dev, d):
    a = np.zeros((8, d), np.float32)
    a[1, d // 2] = np.inf
    a[2, 0] = np.nan
    a[3] = 1.0
    a[4, -1] = -np.inf
    a[4, 0] = np.nan
    a[5] = 2.0 ** -120          # below the smallest amax that gets codes
    a[6, d - 1] = 2.0 ** -100
    a[7] = -5.0
    buf = torch.from_numpy(a).cuda()
    r = x.Rows(ref.F32, buf.data_ptr(), d, None, None)
    q = torch.empty((8, d), dtype=torch.int8, device=dev)
    sc = torch.empty(8, device=dev)
    x.quant_i8(8, d, r, q.data_ptr(), sc.data_ptr(), stream())
    check(q, sc, a, np.ones(8), 8, d)
    assert np.isnan(sc.cpu().numpy()).tolist() == [False, True, True, False, True, False, False, False]
    w = torch.ones(d, device=dev)
    x.add_rmsnorm_i8(8, d, r, None, w.data_ptr(), EPS, None, 0, q.data_ptr(), sc.data_ptr(), stream())
    with np.errstate(all="ignore"):
        f = 1 / np.sqrt((a.astype(np.float64) ** 2).mean(1) + EPS)
    check(q, sc, a, f, 8, d)


def test_many_rows(dev):
    n, d = 70001, 40
    g = np.random.default_rng(1)
    buf, r, vals, keep = make(g, n, d, ref.BF16)
    q = torch.empty((n, d), dtype=torch.int8, device=dev)
    sc = torch.empty(n, device=dev)
    x.quant_i8(n, d, r, q.data_ptr(), sc.data_ptr(), stream())
    check(q, sc, vals, np.ones(n), n, d)
