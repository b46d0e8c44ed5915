"""x100_quant_fp8_hip, x100_add_rmsnorm_fp8_hip and x100_gemm_fp8_hip against their definitions: codes bit for bit, scales
and products within the errors of fp32 sums."""
import numpy as np
import pytest
import torch

import fp8_ref as fr
import paged_ref as ref
import x100hip as x
from test_rows_gpu import make, stream

pytestmark = pytest.mark.gpu

EPS = 1e-6


def check_rows(q, scale, t, factor, d, row_ok=None):
    """q [n, ld] and scale [blocks, lds] (torch) of values t [n, d]; factor fp64 [n]."""
    n = len(t)
    want, amax, ok = fr.codes(t)
    if row_ok is not None:
        ok = ok & row_ok[:, None]
        want = np.where(np.repeat(ok, 128, 1)[:, :want.shape[1]], want, 0)
    got = q.cpu().numpy()[:, :want.shape[1]]
    assert np.array_equal(got, want), np.argwhere(got != want)[:5]
    s = np.where(ok, amax.astype(np.float64) * factor[:, None] / 448, np.nan)
    have = scale.cpu().numpy().astype(np.float64)[:, :n].T
    assert np.array_equal(np.isnan(have), np.isnan(s))
    # fp64 squares; the root, its reciprocal, a product and a quotient in fp32, and fp32's smallest numbers
    bound = np.abs(s) * 8 * 2.0 ** -24 + 2.0 ** -149
    keep = ~np.isnan(s)
    assert (np.abs(have - s)[keep] <= bound[keep]).all()


SIZES = [(1, 1), (3, 7), (2, 8), (5, 64), (2, 120), (2, 127), (2, 128), (3, 129), (4, 511), (4, 512), (3, 513), (7, 520),
         (3, 1000), (2, 2048), (2, 2049), (3, 2056), (2, 4096), (1, 4104), (2, 5000), (1, 8192), (1, 16383), (2, 16384),
         (300, 24), (2051, 136), (2049, 640), (4100, 520)]


@pytest.mark.parametrize("t", [ref.F32, ref.F16, ref.BF16, ref.I32])
@pytest.mark.parametrize("n,d", SIZES)
def test_quant(dev, n, d, t):
    g = np.random.default_rng(n * 100003 + d)
    dp, nb = -(-d // 16) * 16, fr.blocks(d)
    for pad, off, more, lds in ((0, 0, 0, n), (8, 0, 16, n + 3), (3, 1, 5, n + 1)):
        buf, r, vals, keep = make(g, n, d, t, pad, off)
        q = torch.full((n, dp + more), 99, dtype=torch.uint8, device=dev)
        sc = torch.full((nb, lds), 7.0, device=dev)
        x.quant_fp8(n, d, r, x.Fp8(q.data_ptr(), dp + more, sc.data_ptr(), lds), stream())
        torch.cuda.synchronize()
        check_rows(q, sc, vals, np.ones(n), d)
        assert (q[:, dp:] == 99).all() and (sc[:, n:] == 7).all()


@pytest.mark.parametrize("xt", [ref.F32, ref.F16, ref.BF16])
@pytest.mark.parametrize("dt", [None, ref.F32, ref.F16, ref.BF16, ref.I32])
@pytest.mark.parametrize("n,d", [(1, 1), (3, 63), (5, 512), (3, 1030), (4, 2048), (2, 4096), (3, 4099), (2, 8200), (1, 16384),
                                 (2050, 264)])
def test_add_rmsnorm(dev, n, d, xt, dt):
    g = np.random.default_rng(n * 7919 + d)
    w = (1 + 0.3 * g.standard_normal(d)).astype(np.float32)
    dw = torch.from_numpy(w).cuda()
    dp, nb = -(-d // 16) * 16, fr.blocks(d)
    for pad, off, inplace in ((0, 0, False), (0, 0, True), (16, 8, False), (5, 3, True)):
        buf, r, vals, keep = make(g, n, d, xt, pad, off)
        q = torch.full((n, dp + 16), 99, dtype=torch.uint8, device=dev)
        sc = torch.full((nb, n), 7.0, device=dev)
        fq = x.Fp8(q.data_ptr(), dp + 16, sc.data_ptr(), n)
        h, rd, ldh, hp = vals, None, d, None
        if dt is not None:
            dbuf, rd, dvals, dkeep = make(g, n, d, dt, pad, off)
            h = (torch.from_numpy(vals) + torch.from_numpy(dvals)).to(fr.TT[xt])
            if inplace:
                hbuf, hp, ldh = buf, r.p, r.ld
            else:
                hbuf = torch.zeros(n * d, dtype=fr.TT[xt], device=dev)
                hp = hbuf.data_ptr()
        x.add_rmsnorm_fp8(n, d, r, rd, dw.data_ptr(), EPS, hp, ldh, fq, stream())
        torch.cuda.synchronize()
        if dt is not None:
            got = (buf[off:].view(n, d + pad)[:, :d] if inplace else hbuf.view(n, d)).cpu()
            assert torch.equal(got, h)
            h = h.float().numpy()
        f = 1 / np.sqrt((h.astype(np.float64) ** 2).mean(1) + EPS)
        check_rows(q, sc, h * w, f, d)
        assert (q[:, dp:] == 99).all()


def test_rows_not_finite(dev):
    """Blocks of zeros, tiny and huge ones, infinities and NaN: alone, and beside blocks that are fine."""
    n, d = 8, 400
    g = np.random.default_rng(5)
    t = g.standard_normal((n, d)).astype(np.float32)
    t[0, :128] = 0
    t[1, 128:256] = 1e-38
    t[2, 5] = 3.4e38
    t[3, 200] = np.inf
    t[4, 399] = np.nan
    t[5] = 0
    t[6, 256:384] = 2.0 ** -99
    buf = torch.from_numpy(t).cuda()
    r = x.Rows(x.T_F32, buf.data_ptr(), d, None, None)
    for norm in (False, True):
        q = torch.full((n, d), 99, dtype=torch.uint8, device=dev)
        sc = torch.full((4, n), 7.0, device=dev)
        fq = x.Fp8(q.data_ptr(), d, sc.data_ptr(), n)
        if not norm:
            x.quant_fp8(n, d, r, fq, stream())
            torch.cuda.synchronize()
            check_rows(q, sc, t, np.ones(n), d)
            continue
        w = torch.ones(d, device=dev)
        x.add_rmsnorm_fp8(n, d, r, None, w.data_ptr(), 0.0, None, d, fq, stream())
        torch.cuda.synchronize()
        ok = np.isfinite(t).all(1)
        with np.errstate(all="ignore"):
            f = 1 / np.sqrt((t.astype(np.float64) ** 2).mean(1))
        f[5] = 0       # a row of zeros has scale 0 with eps = 0 too
        check_rows(q, sc, t, np.where(ok, f, 0), d, ok)


def operands(g, M, N, K, pad_a=0, pad_w=0, nan=False):
    """Codes over the whole range of e4m3, fp64-checkable scales; device tensors with padded rows of NaN codes."""
    def codes(n, pad):
        c = g.integers(0, 256, (n, K), dtype=np.uint8)
        c = np.where((c & 0x7f) == 0x7f, c - 1, c).astype(np.uint8)
        d = torch.full((n, K + pad), 0x7f, dtype=torch.uint8)
        d[:, :K] = torch.from_numpy(c)
        return c, d.cuda()
    a, da = codes(M, pad_a)
    w, dw = codes(N, pad_w)
    sa = (0.1 + g.random((fr.blocks(K), M))).astype(np.float32) * (1 - 2 * (g.random((fr.blocks(K), M)) < 0.1)).astype(np.float32)
    sw = (0.1 + g.random((fr.blocks(N), fr.blocks(K)))).astype(np.float32)
    return a, da, sa, w, dw, sw


def run_gemm(dev, g, M, N, K, ct, pad_a=0, pad_w=0, pad_c=0, off=0, lds=0):
    a, da, sa, w, dw, sw = operands(g, M, N, K, pad_a, pad_w)
    dsa = torch.full((sa.shape[0], M + lds), float("nan"), device=dev)
    dsa[:, :M] = torch.from_numpy(sa)
    dsw = torch.full((sw.shape[0], sw.shape[1] + lds), float("nan"), device=dev)
    dsw[:, :sw.shape[1]] = torch.from_numpy(sw)
    sa, sw = sa.astype(np.float32), sw
    buf = torch.full((off + M * (N + pad_c),), 77.0, dtype=fr.TT[ct], device=dev)
    scale = 1.0 / 4096 if ct == ref.F16 else 1.0          # products of random codes leave fp16 else
    dsw *= scale
    sw = sw * np.float32(scale)
    fa = x.Fp8(da.data_ptr(), K + pad_a, dsa.data_ptr(), M + lds)
    fw = x.Fp8(dw.data_ptr(), K + pad_w, dsw.data_ptr(), sw.shape[1] + lds)
    x.gemm_fp8(M, N, K, fa, fw, ct, buf.data_ptr() + off * buf.element_size(), N + pad_c, stream())
    torch.cuda.synchronize()
    c, size = fr.product(a, sa, w, sw)
    got = buf[off:].view(M, N + pad_c)
    assert (got[:, N:] == 77).all() and (buf[:off] == 77).all()
    far = np.abs(got[:, :N].double().cpu().numpy() - c)
    bound = fr.product_bound(K, c, size, ct)
    assert (far <= bound).all(), (M, N, K, np.argwhere(far > bound)[:5], (far / bound).max())
    if ct != ref.F32:      # some outputs within what they themselves can lose
        m, n = g.integers(0, M, 1000), g.integers(0, N, 1000)
        near = fr.product_bound(K, c[m, n], size[m, n], ct, fr.group_largest(a, sa, w, sw, m, n))
        assert (far[m, n] <= near).all(), (M, N, K, (far[m, n] / near).max())


GEMM = [(1, 1, 16), (1, 16, 128), (1, 5120, 2048), (3, 17, 48), (2, 130, 144), (5, 257, 1000 // 16 * 16), (8, 1000, 2048),
        (15, 129, 240), (16, 64, 4096), (17, 300, 512), (31, 48, 272), (33, 513, 1040), (64, 256, 128), (64, 2048, 4096),
        (65, 127, 640), (100, 1000, 1008), (127, 129, 112), (128, 128, 128), (129, 255, 2064), (200, 384, 16), (255, 257, 384),
        (256, 256, 256), (257, 513, 2048), (333, 6144, 2048), (511, 640, 144), (600, 520, 1296), (1024, 1024, 512),
        (1000, 96, 4096), (2050, 70, 320), (40, 4000, 7168)]
# every kind of tile, with a short last block, rows and columns that end inside a tile, and groups without a last block
GEMM += [(33, 70, 1808), (18, 33, 656), (64, 4096, 656), (128, 5120, 656), (130, 5100, 400), (17, 64, 400), (300, 5120, 400),
         (130, 5100, 272), (700, 5120, 400), (900, 5130, 1296), (1500, 5120, 400), (2300, 4400, 112), (2048, 5120, 144),
         (2047, 5111, 656), (4100, 4300, 272), (5, 8208, 1040), (16, 9000, 144), (4, 8200, 272), (64, 4200, 1040),
         (200, 1500, 912), (250, 2000, 1808), (60, 5120, 656), (3000, 5120, 144), (2900, 5130, 400), (1550, 5130, 528),
         (3400, 2100, 1040)]


@pytest.mark.parametrize("ct", [ref.F32, ref.F16, ref.BF16])
@pytest.mark.parametrize("M,N,K", GEMM)
def test_gemm(dev, M, N, K, ct):
    run_gemm(dev, np.random.default_rng(M * 7 + N * 3 + K + ct), M, N, K, ct)


@pytest.mark.parametrize("ct", [ref.F32, ref.BF16])
@pytest.mark.parametrize("M,N,K", [(1, 33, 160), (16, 200, 256), (70, 130, 400), (300, 260, 528), (520, 1030, 2048)])
def test_gemm_strides(dev, M, N, K, ct):
    """Rows, scales and outputs further apart than they are long, C at every alignment."""
    for pad_a, pad_w, pad_c, off, lds in ((16, 0, 0, 1, 0), (0, 48, 4, 0, 5), (32, 16, 3, 2, 1), (128, 128, 8, 8, 64)):
        run_gemm(dev, np.random.default_rng(M + off), M, N, K, ct, pad_a, pad_w, pad_c, off, lds)


@pytest.mark.parametrize("M,N,K", [(1, 40, 144), (20, 40, 144), (300, 300, 400)])
def test_gemm_nan(dev, M, N, K):
    """A NaN code or scale reaches its row or column, and nothing else."""
    g = np.random.default_rng(3)
    a, da, sa, w, dw, sw = operands(g, M, N, K)
    m, n = M - 1, N // 2
    da[m, K - 1] = 0x7f
    dw[n, 3] = 0xff
    dsa, dsw = torch.from_numpy(sa).cuda(), torch.from_numpy(sw).cuda()
    c = torch.zeros(M, N, device=dev)
    x.gemm_fp8(M, N, K, x.Fp8(da.data_ptr(), K, dsa.data_ptr(), M), x.Fp8(dw.data_ptr(), K, dsw.data_ptr(), sw.shape[1]),
               x.T_F32, c.data_ptr(), N, stream())
    nan = torch.isnan(c)
    want = torch.zeros(M, N, dtype=torch.bool, device=dev)
    want[m, :] = True
    want[:, n] = True
    assert torch.equal(nan, want)
    da[m, K - 1] = dw[n, 3] = 0
    dsw[0, 1] = float("nan")
    x.gemm_fp8(M, N, K, x.Fp8(da.data_ptr(), K, dsa.data_ptr(), M), x.Fp8(dw.data_ptr(), K, dsw.data_ptr(), sw.shape[1]),
               x.T_F32, c.data_ptr(), N, stream())
    nan = torch.isnan(c)
    assert nan[:, :128].all() and not nan[:, 128:].any()


@pytest.mark.parametrize("M,N,K", [(1, 512, 1024), (48, 512, 1024), (300, 512, 1024)])
def test_same_bits_and_graph(dev, M, N, K):
    """Repeated, on another stream and replayed from a graph with new contents: the same bits."""
    g = np.random.default_rng(8)
    a, da, sa, w, dw, sw = operands(g, M, N, K)
    dsa, dsw = torch.from_numpy(sa).cuda(), torch.from_numpy(sw).cuda()
    fa, fw = x.Fp8(da.data_ptr(), K, dsa.data_ptr(), M), x.Fp8(dw.data_ptr(), K, dsw.data_ptr(), sw.shape[1])
    c = [torch.zeros(M, N, device=dev) for _ in range(3)]
    x.gemm_fp8(M, N, K, fa, fw, x.T_F32, c[0].data_ptr(), N, stream())
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    x.gemm_fp8(M, N, K, fa, fw, x.T_F32, c[1].data_ptr(), N, side.cuda_stream)
    side.synchronize()
    assert torch.equal(c[0], c[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x.gemm_fp8(M, N, K, fa, fw, x.T_F32, c[2].data_ptr(), N, torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        da.copy_(da.flip(0).contiguous())
        graph.replay()
        x.gemm_fp8(M, N, K, fa, fw, x.T_F32, c[0].data_ptr(), N, stream())
        torch.cuda.synchronize()
        assert torch.equal(c[0], c[2])


@pytest.mark.parametrize("ct", [ref.F32, ref.F16, ref.BF16])
@pytest.mark.parametrize("M", [1, 9, 17, 40, 72, 129, 137, 1505, 1537, 2057, 3080, 4097, 6009])
def test_gemm_rows_behind_are_left(dev, M, ct):
    """Rows that end inside every kind of tile: those behind M keep what they held, and the last ones are right."""
    N, K = 5120, 272
    g = np.random.default_rng(M)
    a, da, sa, w, dw, sw = operands(g, M, N, K)
    if ct == ref.F16:
        sw = sw * np.float32(1.0 / 4096)
    dsa, dsw = torch.from_numpy(sa).cuda(), torch.from_numpy(sw).cuda()
    c = torch.full((M + 300, N), 77.0, dtype=fr.TT[ct], device=dev)
    x.gemm_fp8(M, N, K, x.Fp8(da.data_ptr(), K, dsa.data_ptr(), M), x.Fp8(dw.data_ptr(), K, dsw.data_ptr(), sw.shape[1]), ct,
               c.data_ptr(), N, stream())
    assert (c[M:] == 77).all()
    r = slice(max(0, M - 40), M)
    want, size = fr.product(a[r], np.ascontiguousarray(sa[:, r]), w, sw)
    far = np.abs(c[r].double().cpu().numpy() - want)
    assert (far <= fr.product_bound(K, want, size, ct)).all()


@pytest.mark.parametrize("ct", [ref.F16, ref.BF16])
@pytest.mark.parametrize("M,N,K", [(1, 40, 144), (20, 40, 144), (300, 5120, 400), (1500, 5120, 400), (2900, 5120, 400), (6000, 5120, 272)])
def test_gemm_nan_16_bits(dev, M, N, K, ct):
    """A NaN code reaches its row or column, also by the 8-bit instruction, and nothing else."""
    g = np.random.default_rng(4)
    a, da, sa, w, dw, sw = operands(g, M, N, K)
    m, n = M - 1, N // 2
    da[m, K - 1] = 0x7f
    dw[n, 3] = 0xff
    dsa, dsw = torch.from_numpy(sa).cuda(), torch.from_numpy(sw / 4096).cuda()
    c = torch.zeros(M, N, dtype=fr.TT[ct], device=dev)
    x.gemm_fp8(M, N, K, x.Fp8(da.data_ptr(), K, dsa.data_ptr(), M), x.Fp8(dw.data_ptr(), K, dsw.data_ptr(), sw.shape[1]), ct,
               c.data_ptr(), N, stream())
    want = torch.zeros(M, N, dtype=torch.bool, device=dev)
    want[m, :] = True
    want[:, n] = True
    assert torch.equal(torch.isnan(c), want)


def test_a_large_product_captured(dev):
    """The persistent tiles in a graph, replayed over new codes beside eager calls on two streams: the same bits."""
    M, N, K = 6001, 5120, 400
    g = np.random.default_rng(9)
    a, da, sa, w, dw, sw = operands(g, M, N, K)
    dsa, dsw = torch.from_numpy(sa).cuda(), torch.from_numpy(sw).cuda()
    fa, fw = x.Fp8(da.data_ptr(), K, dsa.data_ptr(), M), x.Fp8(dw.data_ptr(), K, dsw.data_ptr(), sw.shape[1])
    c = [torch.zeros(M, N, dtype=torch.bfloat16, device=dev) for _ in range(3)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x.gemm_fp8(M, N, K, fa, fw, x.T_BF16, c[2].data_ptr(), N, torch.cuda.current_stream().cuda_stream)
    side = torch.cuda.Stream()
    for _ in range(3):
        da.copy_(da.flip(0).contiguous())
        torch.cuda.synchronize()
        x.gemm_fp8(M, N, K, fa, fw, x.T_BF16, c[1].data_ptr(), N, side.cuda_stream)
        graph.replay()
        x.gemm_fp8(M, N, K, fa, fw, x.T_BF16, c[0].data_ptr(), N, stream())
        torch.cuda.synchronize()
        assert torch.equal(c[0], c[1]) and torch.equal(c[0], c[2]) and not torch.isnan(c[0]).any()


@pytest.mark.parametrize("ct", [ref.F32, ref.BF16])
@pytest.mark.parametrize("M,N,K", [(6300, 5120, 144), (6301, 5120, 256), (4700, 5120, 144), (4711, 5100, 256), (6090, 4088, 16),
                                   (6081, 4096, 128), (2022, 2048, 112), (751, 5120, 16), (4650, 2048, 384)])
def test_gemm_large_and_short(dev, M, N, K, ct):
    """Large tiles over one to three blocks of k, several tiles to a CU."""
    run_gemm(dev, np.random.default_rng(M + K), M, N, K, ct)


@pytest.mark.parametrize("M,N,K", [(3, 200, 272), (40, 200, 272), (400, 300, 272)])
@pytest.mark.parametrize("ea,ew", [(-63, -62), (100, -100), (-110, 90), (60, 40), (-70, -66)])
def test_gemm_scales_of_any_size(dev, M, N, K, ea, ew):
    """Scales far from 1 whose product is a number of fp32, down to its subnormal ones."""
    g = np.random.default_rng(M)
    a, da, _, w, dw, _ = operands(g, M, N, K)
    sa = np.full((fr.blocks(K), M), 2.0 ** ea, np.float32)
    sw = np.full((fr.blocks(N), fr.blocks(K)), 2.0 ** ew, np.float32)
    dsa, dsw = torch.from_numpy(sa).cuda(), torch.from_numpy(sw).cuda()
    c = torch.zeros(M, N, device=dev)
    x.gemm_fp8(M, N, K, x.Fp8(da.data_ptr(), K, dsa.data_ptr(), M), x.Fp8(dw.data_ptr(), K, dsw.data_ptr(), sw.shape[1]),
               x.T_F32, c.data_ptr(), N, stream())
    want, size = fr.product(a, sa, w, sw)
    # an addition per block may end among fp32's subnormal numbers: a step of these each
    bound = fr.product_bound(K, want, size, ref.F32) + fr.blocks(K) * 2.0 ** -149
    assert (np.abs(c.double().cpu().numpy() - want) <= bound).all()
