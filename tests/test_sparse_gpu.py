"""Sparse attention over the paged cache (x100_sparse.h): block means, selection and attention over lists, against plain
forms in 64 bits (sparse_ref.py)."""
import numpy as np
import pytest
import torch

import paged_ref as ref
import sparse_ref as sp
import x100hip as x
from test_paged_gpu import Setup, TT, compare, dev_i32, kinds, stream

pytestmark = pytest.mark.gpu


def rows_of(t):
    return list(sp.rows_of(t.q_start, t.kv_lens, t.n_rows, t.max_q, t.max_kv))


def lists(t, n_sel, g, own_share=0.8):
    """Random ascending lists: most end at the row's own block, some are short, some empty."""
    c = t.c
    sel = np.full((t.n_rows, c.n_kv, n_sel), -1, np.int64)
    for r, s, pos in rows_of(t):
        own = pos // c.page if pos >= 0 else -1
        for h in range(c.n_kv):
            n = min(n_sel, own + 1)
            if g.random() < 0.2:
                n = int(g.integers(0, n + 1))
            pick = g.permutation(own + 1)[:n]
            if n and g.random() < own_share and own not in pick:
                pick[0] = own
            sel[r, h, :n] = np.sort(pick)
    return sel


def attend(t, dq, ldq, sel, n_sel, scale, ws=True, ldo=None, out=None, st=None):
    c = t.c
    ldo = ldo or c.n_head * c.hd
    if out is None:
        out = torch.full((t.n_rows, ldo), -7.0, dtype=TT[c.act], device="cuda")
    a = (t.cfg, t.batch, dq.data_ptr(), ldq, t.dk.data_ptr(), t.dv.data_ptr(), scale, sel.data_ptr(), n_sel, out.data_ptr(), ldo)
    st = stream() if st is None else st
    if ws:
        n = x.attn_sparse_workspace_bytes(t.cfg, t.batch, n_sel)
        w = torch.full((max(n, 256),), 255, dtype=torch.uint8, device="cuda")
        x.attn_sparse_ws(*a, w.data_ptr(), n, st)
        torch.cuda.synchronize()
    else:
        x.attn_sparse(*a, st)
        torch.cuda.synchronize()
    return out


def check(t, n_sel, sel=None, gain=1.0, pad=0, ws=True):
    c = t.c
    if sel is None:
        sel = lists(t, n_sel, t.g)
    dq, q = t.queries(gain, pad)
    scale = c.hd ** -0.5
    out = attend(t, dq, c.n_head * c.hd + pad, dev_i32(sel), n_sel, scale, ws)
    K, V = c.decode(t.kb, t.vb)
    want = np.full((t.n_rows, c.n_head, c.hd), -7.0)
    tol = sp.attend(c, K, V, q, rows_of(t), t.table, sel, scale, want)
    compare(out.float().cpu().numpy().astype(np.float64).reshape(want.shape), want, tol)
    return out, dq, sel


# ---- attention over lists -----------------------------------------------------------------------
@kinds
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("page", [16, 64])
def test_single_tokens(dev, act, kv, hd, page):
    lens = [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 300, 500]
    for n_sel in (1, 3, 8):
        check(Setup(1, 8, 2, hd, page, act, kv, [1] * len(lens), lens), n_sel)


@kinds
@pytest.mark.parametrize("n_head,n_kv", [(1, 1), (4, 4), (6, 2), (5, 1), (16, 1), (14, 2), (9, 3)])
def test_head_groups(dev, act, kv, n_head, n_kv):
    check(Setup(2, n_head, n_kv, 128, 32, act, kv, [1, 3, 1, 6], [40, 3, 200, 177]), 4)


@kinds
@pytest.mark.parametrize("page", [16, 32, 128, 256])
def test_prompts(dev, act, kv, page):
    check(Setup(3, 4, 2, 128, page, act, kv, [1, 2, 17, 40, 33], [1, 2, 17, 400, 900]), 3)


@kinds
@pytest.mark.parametrize("kv_len,n_sel", [(1000, 40), (3000, 47), (2049, 129), (5000, 512)])
def test_splits(dev, act, kv, kv_len, n_sel):
    """Few rows and long lists: the list's positions in many parts, joined; some parts have nothing."""
    t = Setup(4, 4, 1, 64, 16, act, kv, [1, 2], [kv_len, kv_len // 3])
    out, dq, sel = check(t, n_sel)
    assert x.attn_sparse_workspace_bytes(t.cfg, t.batch, n_sel) > 0
    again = attend(t, dq, 4 * 64, dev_i32(sel), n_sel, 64 ** -0.5, ws=False)
    assert torch.equal(out, again)


@kinds
def test_all_blocks_is_the_dense_attention(dev, act, kv):
    t = Setup(5, 8, 2, 128, 32, act, kv, [1, 5, 20], [300, 170, 20])
    n_sel = 12
    sel = np.full((t.n_rows, 2, n_sel), -1, np.int64)
    for r, s, pos in rows_of(t):
        sel[r, :, :pos // 32 + 1] = np.arange(pos // 32 + 1)
    dq, q = t.queries()
    out = attend(t, dq, 1024, dev_i32(sel), n_sel, 128 ** -0.5)
    want, tol = t.expected(q, 128 ** -0.5)
    compare(out.float().cpu().numpy().astype(np.float64).reshape(want.shape), want, tol)


@kinds
def test_broken_lists_and_pages(dev, act, kv):
    """Entries that are out of order, behind the own block or below 0 end a list; blocks without a page are skipped."""
    t = Setup(6, 4, 2, 64, 16, act, kv, [1] * 9 + [3], [160] * 9 + [40])
    own = 9
    sel = np.full((t.n_rows, 2, 6), -1, np.int64)
    bad = [[3, 3, 4, 5, 6, 9], [9, 2, 9, 1, 9, 9], [1, 10, 2, 3, 4, 9], [-5, 1, 2, 3, 4, 9], [0, 2, 4, 6, 8, 9],
           [2, 1 << 30, 3, 4, 5, 6], [7, 8, 9, 9, 9, 9], [-1] * 6, [own, own + 1, 3, 2, 1, 0]]
    for i, b in enumerate(bad):
        sel[i, 0] = b
        sel[i, 1] = b[::-1]
    sel[9:, :, 0] = [[0], [1], [2]]
    t.table[4, 2], t.table[4, 9], t.table[0, 3] = -1, t.c.n_pages, 1 << 30
    t.upload()
    check(t, 6, sel)


@kinds
def test_not_finite(dev, act, kv):
    """Infinities and NaN in blocks that a list names reach the row, those elsewhere and behind the row's position do not."""
    t = Setup(7, 4, 1, 64, 16, act, kv, [1, 2, 1], [100, 90, 64])
    K, V = t.c.decode(t.kb, t.vb)
    big = np.inf if kv != ref.Q4 else np.nan
    K[t.table[0, 1], 0, 3, 5] = np.nan
    V[t.table[1, 2], 0, 4, 7] = big
    V[t.table[2, 0], 0, 15, 1] = -big
    K[t.table[1, 3]] = np.nan
    with np.errstate(invalid="ignore"):
        t.kb, t.vb = t.c.encode(K.astype(np.float32), V.astype(np.float32))
    t.upload()
    sel = np.full((4, 1, 4), -1, np.int64)
    sel[0, 0, :3] = [0, 1, 6]
    sel[1, 0, :3] = [0, 2, 5]
    sel[2, 0, :3] = [0, 1, 5]
    sel[3, 0, :2] = [1, 3]
    out, dq, _ = check(t, 4, sel)
    o = out.float().view(4, 4, 64)
    assert torch.isnan(o[0]).all() and torch.isfinite(o[2:]).all()


@kinds
def test_rows_before_the_first_position(dev, act, kv):
    t = Setup(8, 4, 2, 64, 16, act, kv, [5, 4, 0, 3], [2, 0, 30, 50], max_q=6, max_kv=64, tail_rows=2)
    check(t, 3)


def test_broken_batches(dev):
    """Sequences that break the bounds: nothing of theirs is written."""
    t = Setup(9, 4, 2, 64, 16, ref.BF16, ref.BF16, [1, 2, 1, 1], [40, 50, 60, 70], max_q=2, max_kv=64)
    sel = lists(Setup(9, 4, 2, 64, 16, ref.BF16, ref.BF16, [1, 2, 1, 1], [40, 50, 60, 64], max_q=2, max_kv=64), 3, t.g)
    check(t, 3, sel)                                     # 70 > max_kv: refused
    t.kv_lens[1] = -3
    t.upload()
    check(t, 3, sel)
    t.kv_lens[1], t.q_start[4] = 50, 9                   # rows behind n_rows
    t.upload()
    check(t, 3, sel)


def test_strides_and_fp32_range_of_queries(dev):
    t = Setup(10, 6, 2, 128, 64, ref.BF16, ref.Q4, [1, 7], [700, 300])
    check(t, 4, pad=64)
    for gain in (1e-6, 30.0):
        check(t, 4, gain=gain)


# ---- means ----------------------------------------------------------------------------------------
@kinds
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 64, 256])
def test_means(dev, act, kv, hd, page):
    t = Setup(11, 4, 3 if hd == 64 else 1, hd, page, act, kv, [1, 1, 1, 3 * page, page + 5, 7, 1, 40],
              [page, page - 1, 2 * page, 3 * page, 2 * page + 5, 3, 5 * page, 4 * page], tail_rows=3) \
        if hd == 128 else Setup(11, 3, 3, hd, page, act, kv, [1, 2 * page + 1, 1, 17], [page, 2 * page + 1, 3 * page, page + 16])
    t.table[0, 0] = -1
    t.upload()
    c = t.c
    old = np.full((c.n_pages, c.n_kv, hd), 0x1234, np.uint16)
    d = torch.from_numpy(old.view(np.int16)).cuda()
    assert x.kv_means_bytes(t.cfg) == old.nbytes
    x.kv_means(t.cfg, t.batch, t.dk.data_ptr(), d.data_ptr(), stream())
    torch.cuda.synchronize()
    K, _ = c.decode(t.kb, t.vb)
    want = sp.means(c, K, rows_of(t), t.table, old)
    assert (want != old).any()
    assert np.array_equal(d.cpu().numpy().view(np.uint16), want)


def test_means_not_finite(dev):
    t = Setup(12, 2, 1, 64, 16, ref.F16, ref.F16, [1, 1], [32, 16])
    K, V = t.c.decode(t.kb, t.vb)
    K[t.table[0, 1], 0, 3, 5], K[t.table[0, 1], 0, 4, 6], K[t.table[1, 0], 0, 0, 0] = np.inf, np.nan, 65504
    K[t.table[1, 0], 0, 1:, 0] = 65504
    with np.errstate(invalid="ignore"):
        t.kb, t.vb = t.c.encode(K.astype(np.float32), V.astype(np.float32))
    t.upload()
    d = torch.zeros(t.c.n_pages, 64, dtype=torch.float16, device=dev)
    x.kv_means(t.cfg, t.batch, t.dk.data_ptr(), d.data_ptr(), stream())
    got = d.cpu().numpy()
    a, b = got[t.table[0, 1]], got[t.table[1, 0]]
    assert a[5] == np.inf and np.isnan(a[6]) and np.isfinite(np.delete(a, [5, 6])).all() and b[0] == 65504


# ---- selection ------------------------------------------------------------------------------------
class Pick:
    """A batch, its page table and random means; the cache itself is not looked at."""

    def __init__(self, seed, n_head, n_kv, hd, page, act, q_lens, kv_lens, tail_rows=0, max_q=None, max_kv=None):
        g = self.g = np.random.default_rng(seed)
        self.q_lens, self.kv_lens = list(q_lens), list(kv_lens)
        self.max_q, self.max_kv = max_q or max(1, max(q_lens)), max_kv or max(1, max(kv_lens))
        per = -(-self.max_kv // page) + 1
        need = [-(-max(n, 0) // page) for n in kv_lens]
        self.c = ref.Cache(n_head, n_kv, hd, page, sum(need) + 1, act, act)
        self.cfg = x.KvCfg(n_head, n_kv, hd, page, self.c.n_pages, act, act)
        self.table = np.full((len(kv_lens), per), -1, np.int64)
        free = list(g.permutation(self.c.n_pages))
        for s, n in enumerate(need):
            for i in range(n):
                self.table[s, i] = free.pop()
        self.q_start = np.concatenate([[0], np.cumsum(q_lens)])
        self.n_rows = int(self.q_start[-1]) + tail_rows
        self.mean = ref.to_bits(g.standard_normal((self.c.n_pages, n_kv, hd)).astype(np.float32), act)
        self.qbits = ref.to_bits(g.standard_normal((self.n_rows, n_head * hd)).astype(np.float32), act)

    def run(self, n_sel, n_first, n_last, st=None):
        self.keep = [dev_i32(self.q_start), dev_i32(self.kv_lens), dev_i32(self.table),
                     torch.from_numpy(self.mean.view(np.int16)).cuda(), torch.from_numpy(self.qbits.view(np.int16)).cuda()]
        qs, kl, tab, m, q = (k.data_ptr() for k in self.keep)
        self.batch = x.KvBatch(len(self.kv_lens), self.n_rows, self.max_q, self.max_kv, self.table.shape[1], qs, kl, tab)
        sel = torch.full((self.n_rows, self.c.n_kv, n_sel), -99, dtype=torch.int32, device="cuda")
        x.attn_select(self.cfg, self.batch, x.KvSel(n_sel, n_first, n_last), q, self.c.n_head * self.c.hd, m, sel.data_ptr(), stream())
        torch.cuda.synchronize()
        return sel.cpu().numpy()

    def check(self, n_sel, n_first=1, n_last=1):
        c = self.c
        got = self.run(n_sel, n_first, n_last)
        want = np.full(got.shape, -99)
        q = ref.from_bits(self.qbits, c.act).reshape(self.n_rows, c.n_head, c.hd)
        rows = list(sp.rows_of(self.q_start, self.kv_lens, self.n_rows, self.max_q, self.max_kv))
        sp.select(c, q, ref.from_bits(self.mean, c.act).reshape(c.n_pages, c.n_kv, c.hd), rows, self.table, n_sel, n_first, n_last, want)
        assert np.array_equal(got, want), np.argwhere((got != want).any(-1))[:5]
        return got


acts = pytest.mark.parametrize("act", [ref.F16, ref.BF16], ids=["f16", "bf16"])


@acts
@pytest.mark.parametrize("hd,n_head,n_kv", [(64, 8, 2), (128, 6, 3), (128, 16, 1), (64, 5, 5)])
def test_select_single_tokens(dev, act, hd, n_head, n_kv):
    lens = [1, 15, 16, 17, 32, 33, 100, 255, 256, 257, 1000, 5000]
    for n_sel, first, last in ((1, 0, 1), (3, 1, 1), (8, 2, 3), (32, 0, 1), (5, 0, 5), (6, 4, 2)):
        Pick(n_sel, n_head, n_kv, hd, 16, act, [1] * len(lens), lens).check(n_sel, first, last)


@acts
@pytest.mark.parametrize("page", [16, 64, 256])
def test_select_prompts(dev, act, page):
    Pick(3, 8, 2, 128, page, act, [1, 5, 40, 17, 3, 70], [900, 5, 400, 1117, 3, 70]).check(4)
    Pick(4, 4, 1, 64, page, act, [9, 6], [page * 100, page * 90 + 3]).check(16, 1, 2)


@acts
@pytest.mark.parametrize("blocks,q", [(1024, 1), (1025, 1), (2500, 5), (4096, 4), (4097, 4), (16384, 1)])
def test_select_many_blocks(dev, act, blocks, q):
    """Every size of the keys' space in LDS, at and beside its end."""
    Pick(5, 2, 1, 64, 16, act, [q, 1], [16 * blocks, 16 * blocks // 3]).check(64, 1, 2)
    Pick(6, 2, 1, 64, 16, act, [q], [16 * blocks - 7]).check(512, 0, 1)


def test_select_ties_and_odd_scores(dev):
    """Equal scores go to the lower block; NaN and -infinity rank last, +infinity first, behind no block that is always taken."""
    p = Pick(7, 4, 2, 64, 16, ref.F16, [1, 1, 1, 1, 6], [640, 640, 640, 640, 640])
    m = p.mean.reshape(p.c.n_pages, 2, 64)
    m[p.table[0, 5:20]] = m[p.table[0, 5]]
    m[p.table[1, :40]] = 0
    m[p.table[1, 3:30:2], :, 0] = 0x8000                    # -0
    m[p.table[2, 4], :, 3], m[p.table[2, 9], :, 3], m[p.table[2, 11], :, 3] = 0x7c00, 0xfc00, 0x7e00
    m[p.table[4, :39]] = 0x7e00
    for n_sel, first, last in ((4, 0, 1), (9, 1, 1), (20, 1, 2), (39, 0, 1), (40, 1, 1)):
        p.check(n_sel, first, last)


def test_select_blocks_without_a_page(dev):
    p = Pick(8, 4, 2, 64, 16, ref.BF16, [1, 1, 5, 1], [640, 300, 320, 64])
    p.table[0, 3:30] = -1
    p.table[1, 5] = p.c.n_pages
    p.table[1, 18] = 1 << 30                                # the own block
    p.table[2, 0] = -7
    p.table[3, :4] = -1                                     # all
    for n_sel, first, last in ((4, 1, 1), (16, 1, 2), (40, 0, 1)):
        p.check(n_sel, first, last)


def test_select_bounds(dev):
    """Rows before position 0 have empty lists; rows of no sequence, and of refused ones, are left."""
    p = Pick(9, 2, 1, 64, 16, ref.BF16, [5, 4, 0, 3], [2, 0, 30, 50], tail_rows=3, max_q=6, max_kv=64)
    got = p.check(3)
    assert (got[-3:] == -99).all() and (got[0] == -1).all()
    for bad in ((1, 70), (1, -1), (3, 65)):
        p.kv_lens[bad[0]] = bad[1]
        p.check(3)
    p.q_start[2] = 20
    p.check(3)


# ---- together -------------------------------------------------------------------------------------
def test_streams_and_graph(dev):
    """Means, selection and attention captured once, replayed over other lengths, keys and queries: as called one by one."""
    t = Setup(13, 8, 2, 64, 16, ref.BF16, ref.BF16, [1, 1, 3], [400, 160, 333], max_kv=512)
    c, n_sel = t.c, 8
    t.dk.view(torch.bfloat16)[:] = torch.randn(t.dk.numel() // 2, device=dev).bfloat16()
    t.dv.view(torch.bfloat16)[:] = torch.randn(t.dv.numel() // 2, device=dev).bfloat16()
    t.d_tab.clamp_(min=0)
    dq, _ = t.queries()
    ws = torch.zeros(max(256, x.attn_sparse_workspace_bytes(t.cfg, t.batch, n_sel)), dtype=torch.uint8, device=dev)
    pick = x.KvSel(n_sel, 1, 2)

    def fresh():
        return (torch.zeros(c.n_pages, 2, 64, dtype=torch.bfloat16, device=dev),
                torch.full((t.n_rows, 2, n_sel), -1, dtype=torch.int32, device=dev),
                torch.zeros(t.n_rows, 512, dtype=torch.bfloat16, device=dev))

    def step(b, st, w):
        x.kv_means(t.cfg, t.batch, t.dk.data_ptr(), b[0].data_ptr(), st)
        x.attn_select(t.cfg, t.batch, pick, dq.data_ptr(), 512, b[0].data_ptr(), b[1].data_ptr(), st)
        x.attn_sparse_ws(t.cfg, t.batch, dq.data_ptr(), 512, t.dk.data_ptr(), t.dv.data_ptr(), 0.125, b[1].data_ptr(), n_sel,
                         b[2].data_ptr(), 512, w.data_ptr(), w.numel(), st)

    one, two = fresh(), fresh()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step(one, torch.cuda.current_stream().cuda_stream, ws)
    side, ws2 = torch.cuda.Stream(), torch.zeros_like(ws)
    for n in ([400, 160, 333], [401, 176, 336], [5, 512, 352], [416, 0, 2]):
        t.d_kl.copy_(dev_i32(n))
        dq.copy_(torch.randn(t.n_rows, 512, device=dev).bfloat16().view(torch.int16))
        torch.cuda.synchronize()
        graph.replay()
        step(two, side.cuda_stream, ws2)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(one, two))


def test_half_layer(dev):
    """The attention half of a layer as a server runs it, in 8-bit floating point and with lists: norm, projections, append,
    means, selection, attention, output projection, the next norm.  Against 64 bits, step by step from what the kernels stored."""
    import fp8_ref as fr
    g = np.random.default_rng(14)
    d, nh, kv, hd, page, n_sel = 512, 8, 2, 64, 16, 6
    q_lens, kv_lens = [1, 33, 1, 16], [200, 150, 97, 16]
    t = Setup(14, nh, kv, hd, page, ref.BF16, ref.BF16, q_lens, kv_lens)
    n, wide = t.n_rows, (nh + 2 * kv) * hd
    kb, vb = t.c.decode(t.kb, t.vb)

    def weights(N, K):
        c = g.integers(0, 256, (N, K), dtype=np.uint8)
        c = np.where((c & 0x7f) > 0x6f, c & 0x8f, c).astype(np.uint8)
        s = (g.random((fr.blocks(N), fr.blocks(K))) / 300 + 1e-4).astype(np.float32)
        dc, ds = torch.from_numpy(c).cuda(), torch.from_numpy(s).cuda()
        return c, s, x.Fp8(dc.data_ptr(), K, ds.data_ptr(), s.shape[1]), (dc, ds)

    def codes(n, K):
        c, s = torch.zeros(n, K, dtype=torch.uint8, device=dev), torch.zeros(fr.blocks(K), n, device=dev)
        return c, s, x.Fp8(c.data_ptr(), K, s.data_ptr(), n)

    def host(v):
        return v.double().cpu().numpy()

    st = stream()
    wq, sq, fq, k1 = weights(wide, d)
    wo, so, fo, k2 = weights(d, nh * hd)
    h = torch.randn(n, d, device=dev).bfloat16()
    w1 = 1 + 0.1 * torch.randn(d, device=dev)
    a8, as_, fa = codes(n, d)
    x.add_rmsnorm_fp8(n, d, x.Rows(x.T_BF16, h.data_ptr(), d, None, None), None, w1.data_ptr(), 1e-6, None, d, fa, st)
    qkv = torch.zeros(n, wide, dtype=torch.bfloat16, device=dev)
    x.gemm_fp8(n, wide, d, fa, fq, x.T_BF16, qkv.data_ptr(), wide, st)
    qkv /= 16                                             # scores of an ordinary size
    rope = torch.zeros(256, hd // 2, 2, device=dev)
    x.rope_table(hd, 256, 1e4, rope.data_ptr(), st)
    part = lambda i: x.Rows(x.T_BF16, qkv.data_ptr() + 2 * i, wide, None, None)  # noqa: E731
    rows = x.KvRows(part(0), part(nh * hd), part((nh + kv) * hd), None, None, 1e-6, rope.data_ptr(), 256)
    dq = torch.zeros(n, nh * hd, dtype=torch.bfloat16, device=dev)
    x.kv_append(t.cfg, t.batch, rows, t.dk.data_ptr(), t.dv.data_ptr(), dq.data_ptr(), st)
    # the pages before the batch's rows were completed by earlier steps: a batch of whole sequences makes their means
    whole = x.KvBatch(len(kv_lens), sum(kv_lens), 256, t.max_kv, t.table.shape[1], 0, t.d_kl.data_ptr(), t.d_tab.data_ptr())
    all_start = dev_i32(np.concatenate([[0], np.cumsum(kv_lens)]))
    whole.q_start = all_start.data_ptr()
    means = torch.zeros(t.c.n_pages, kv, hd, dtype=torch.bfloat16, device=dev)
    x.kv_means(t.cfg, whole, t.dk.data_ptr(), means.data_ptr(), st)
    sel = torch.zeros(n, kv, n_sel, dtype=torch.int32, device=dev)
    x.attn_select(t.cfg, t.batch, x.KvSel(n_sel, 1, 2), dq.data_ptr(), nh * hd, means.data_ptr(), sel.data_ptr(), st)
    o = torch.zeros(n, nh * hd, dtype=torch.bfloat16, device=dev)
    x.attn_sparse(t.cfg, t.batch, dq.data_ptr(), nh * hd, t.dk.data_ptr(), t.dv.data_ptr(), 0.125, sel.data_ptr(), n_sel,
                  o.data_ptr(), nh * hd, st)
    o8, os_, fo8 = codes(n, nh * hd)
    x.quant_fp8(n, nh * hd, x.Rows(x.T_BF16, o.data_ptr(), nh * hd, None, None), fo8, st)
    y = torch.zeros(n, d, dtype=torch.bfloat16, device=dev)
    x.gemm_fp8(n, d, nh * hd, fo8, fo, x.T_BF16, y.data_ptr(), d, st)
    h0 = h.clone()
    hx = x.Rows(x.T_BF16, h.data_ptr(), d, None, None)
    x.add_rmsnorm_fp8(n, d, hx, x.Rows(x.T_BF16, y.data_ptr(), d, None, None), w1.data_ptr(), 1e-6, h.data_ptr(), d, fa, st)
    torch.cuda.synchronize()

    c, size = fr.product(o8.cpu().numpy(), os_.cpu().numpy(), wo, so)
    assert (np.abs(host(y) - c) <= fr.product_bound(nh * hd, c, size, ref.BF16)).all()
    assert torch.equal(h, (h0.float() + y.float()).bfloat16())
    K, V = t.c.decode(t.dk.cpu().numpy(), t.dv.cpu().numpy())
    rr = rows_of(t)
    want = np.zeros((n, kv, n_sel), np.int64)
    q = host(dq).reshape(n, nh, hd)
    old = np.zeros((t.c.n_pages, kv, hd), np.uint16)
    wm = sp.means(t.c, K, list(sp.rows_of(np.concatenate([[0], np.cumsum(kv_lens)]), kv_lens, sum(kv_lens), 256, 256)), t.table, old)
    assert np.array_equal(means.cpu().view(torch.int16).numpy().view(np.uint16), wm)
    sp.select(t.c, q, host(means), rr, t.table, n_sel, 1, 2, want)
    assert np.array_equal(sel.cpu().numpy(), want)
    out = np.zeros((n, nh, hd))
    tol = sp.attend(t.c, K, V, q, rr, t.table, want, 0.125, out)
    compare(host(o).reshape(n, nh, hd), out, tol)


def test_select_under_wide_bounds(dev):
    """Single tokens and prompts under bounds that any of them may reach, as a captured graph has them."""
    for q_lens, rows_more in (([1, 1, 1], 0), ([1, 20, 7], 0), ([8, 9, 1], 12), ([3, 3, 3, 40, 1, 8], 100)):
        n = len(q_lens)
        for max_q in (40, 300):
            p = Pick(20, 4, 2, 64, 16, ref.BF16, q_lens, [700, 650, 300, 900, 16, 100][:n], tail_rows=rows_more, max_q=max_q, max_kv=2000)
            p.check(6, 1, 2)
            p = Pick(21, 4, 2, 64, 16, ref.BF16, q_lens, [700, 650, 300, 900, 16, 100][:n], tail_rows=n * max_q - sum(q_lens),
                     max_q=max_q, max_kv=1000)
            p.check(6, 1, 2)


def test_select_and_means_of_many_sequences(dev):
    """More sequences than a wave looks at together, most of them without rows."""
    q_lens = ([0] * 70 + [1] + [0] * 3 + [2]) * 4 + [1] * 40
    kv_lens = [16 * (i % 7 + 1) for i in range(len(q_lens))]
    p = Pick(22, 2, 1, 64, 16, ref.F16, q_lens, kv_lens)
    p.check(3)
    t = Setup(23, 2, 1, 64, 16, ref.F16, ref.F16, q_lens, kv_lens)
    d = torch.zeros(t.c.n_pages, 1, 64, dtype=torch.int16, device=dev)
    x.kv_means(t.cfg, t.batch, t.dk.data_ptr(), d.data_ptr(), stream())
    torch.cuda.synchronize()
    K, _ = t.c.decode(t.kb, t.vb)
    want = sp.means(t.c, K, rows_of(t), t.table, np.zeros((t.c.n_pages, 1, 64), np.uint16))
    assert np.array_equal(d.cpu().numpy().view(np.uint16), want)


def test_means_of_refused_sequences(dev):
    """A sequence that breaks its bounds between others: theirs are made, its own and no other page is touched."""
    t = Setup(24, 2, 1, 64, 16, ref.BF16, ref.BF16, [1, 17, 1, 16, 1], [32, 48, 64, 80, 16], max_q=16, max_kv=80)
    old = np.full((t.c.n_pages, 1, 64), 0x77, np.uint16)
    d = torch.from_numpy(old.view(np.int16).copy()).cuda()
    x.kv_means(t.cfg, t.batch, t.dk.data_ptr(), d.data_ptr(), stream())
    torch.cuda.synchronize()
    K, _ = t.c.decode(t.kb, t.vb)
    want = sp.means(t.c, K, rows_of(t), t.table, old)
    assert len(rows_of(t)) == 19 and np.array_equal(d.cpu().numpy().view(np.uint16), want)


@acts
def test_select_prompts_ties_and_odd_scores(dev, act):
    """As test_select_ties_and_odd_scores and the blocks without a page, for rows that are taken together."""
    inf = 0x7c00 if act == ref.F16 else 0x7f80
    for seed, n_head, n_kv, hd in ((30, 4, 2, 64), (31, 3, 1, 128)):
        p = Pick(seed, n_head, n_kv, hd, 16, act, [20, 17, 8, 33, 40], [640, 300, 900, 33, 560])
        m = p.mean.reshape(p.c.n_pages, n_kv, hd)
        m[p.table[0, 5:20]] = m[p.table[0, 5]]
        m[p.table[1, :18]] = 0
        m[p.table[1, 3:15:2], :, 0] = 0x8000
        m[p.table[2, 4], :, 3], m[p.table[2, 9], :, 3], m[p.table[2, 11], :, 3] = inf, inf | 0x8000, inf | 0x200
        m[p.table[4, :30]] = inf | 0x200
        p.table[2, 20:40] = -1
        p.table[3, 0] = p.c.n_pages
        p.table[4, 32] = 1 << 30
        for n_sel, first, last in ((1, 0, 1), (4, 0, 1), (5, 2, 3), (9, 1, 1), (20, 1, 2), (39, 0, 1), (40, 1, 1), (64, 30, 34)):
            p.check(n_sel, first, last)


@acts
def test_select_prompts_of_close_scores(dev, act):
    """Scores that share their upper bits: all digits of the keys are needed."""
    p = Pick(32, 2, 1, 64, 16, act, [24], [1600])
    m = p.mean.reshape(p.c.n_pages, 64)
    base = m[p.table[0, 0]].copy()
    for i in range(100):
        m[p.table[0, i]] = base
        m[p.table[0, i], 7] = (0x0001 if act == ref.F16 else 0x2000) + i % 23      # tiny next to the others
    for n_sel in (3, 10, 50):
        p.check(n_sel, 0, 1)
    p.q_start, p.q_lens, p.kv_lens, p.n_rows, p.max_q = np.array([0, 1]), [1], [1600], 1, 1
    p.qbits = p.qbits[:1]
    for n_sel in (3, 10, 50):
        p.check(n_sel, 0, 1)


def test_select_of_more_blocks_than_a_launch_holds(dev):
    """4097 rows by 1024 KV heads, with tables of more than 1024 pages: 2^22 + 2^10 lists of blocks of 1024 threads."""
    n, nh, pages = 4097, 1024, 3
    g = np.random.default_rng(27)
    cfg = x.KvCfg(nh, nh, 64, 16, pages, x.T_BF16, x.T_BF16)
    kv_lens = g.integers(1, 49, n)
    table = np.full((n, 1025), -1)
    table[:, :3] = np.argsort(g.random((n, 3)), axis=1)
    torch.manual_seed(27)
    q = torch.randn(n, nh, 64, dtype=torch.bfloat16, device=dev)
    means = torch.randn(pages, nh, 64, dtype=torch.bfloat16, device=dev)
    sel = torch.full((n, nh, 2), -99, dtype=torch.int32, device=dev)
    qs, kl, tab = dev_i32(np.arange(n + 1)), dev_i32(kv_lens), dev_i32(table)
    b = x.KvBatch(n, n, 1, 16 * 1025, 1025, qs.data_ptr(), kl.data_ptr(), tab.data_ptr())
    x.attn_select(cfg, b, x.KvSel(2, 0, 1), q.data_ptr(), nh * 64, means.data_ptr(), sel.data_ptr(), stream())
    torch.cuda.synchronize()
    # of blocks 0 and 1 the better one, where the row's own is 2
    better = torch.empty(n, nh, dtype=torch.int32, device=dev)
    for r in range(0, n, 512):
        pg = tab[r:r + 512, :2].long()
        y = [(q[r:r + 512].double() * means[pg[:, i]].double()).sum(-1) for i in (0, 1)]
        better[r:r + 512] = (y[1] > y[0]).int()
    own = dev_i32((kv_lens - 1) // 16)[:, None].expand(n, nh)
    zero = torch.zeros_like(better)
    want = torch.stack([torch.where(own == 2, better, zero), torch.where(own == 0, zero - 1, own)], -1)
    assert torch.equal(sel, want)


@acts
@pytest.mark.parametrize("blocks", [40, 1500, 3000, 5000])
def test_select_few_sequences_under_wide_bounds(dev, act, blocks):
    """Prompts and single tokens of few sequences, some empty, refused or before position 0, in a batch of many rows."""
    kv = 16 * blocks
    q_lens = [1, 9, 0, 7, 30, 2, 8, 20, 5, 1]
    kv_lens = [kv, kv - 5, 33, 300, kv - 17, -1, 5, kv + 1, 3, 170]
    p = Pick(28, 4, 2, 64, 16, act, q_lens, kv_lens, tail_rows=30, max_q=25, max_kv=kv)
    got = p.check(6, 1, 2)
    first = [int(n) for n in p.q_start]
    assert (got[first[4]:first[5]] == -99).all()          # 30 rows > max_q
    assert (got[first[5]:first[6]] == -99).all() and (got[first[7]:first[8]] == -99).all()
    assert (got[first[6]:first[6] + 3] == -1).all() and (got[first[8]:first[8] + 2] == -1).all()
    assert (got[first[-1]:] == -99).all()


@acts
@pytest.mark.parametrize("blocks", [1100, 2100])
def test_select_prompts_of_many_blocks_with_ties(dev, act, blocks):
    """Equal scores, scores that share their upper bits, and blocks without a page, on long contexts."""
    p = Pick(33, 4, 2, 64, 16, act, [18, 9], [16 * blocks, 16 * blocks - 100])
    m = p.mean.reshape(p.c.n_pages, 2, 64)
    m[p.table[0, 100:900]] = m[p.table[0, 100]]
    base = m[p.table[1, 0]].copy()
    for i in range(1000):
        m[p.table[1, i]] = base
        m[p.table[1, i], :, 7] = (0x0001 if act == ref.F16 else 0x2000) + i % 23      # tiny next to the others
    p.table[1, 1000:blocks - 7] = -1
    for n_sel, first, last in ((3, 0, 1), (60, 1, 2), (300, 0, 1), (512, 2, 2)):
        p.check(n_sel, first, last)
    p.qbits[:] = 0
    p.check(40, 1, 1)


@acts
@pytest.mark.parametrize("blocks", [30, 600, 1100, 2100])
@pytest.mark.parametrize("score", [-1.0, -2.0, 2.0 - 2.0 ** -24, "one"])
def test_select_of_forced_blocks_alone(dev, act, blocks, score):
    """Lists that the first and last blocks fill, on prompts and single rows, where the other blocks' scores have keys that end in
    ones: no other block is listed, and nothing behind the lists is written."""
    p = Pick(34, 4, 2, 64, 16, act, [21, 1, 9], [16 * blocks, 16 * blocks - 9, 16 * blocks - 40], tail_rows=5)
    q = np.zeros((p.n_rows, 4, 64))
    q[:, :, :2] = 0.5                                      # two heads: sums of 1
    p.qbits = ref.to_bits(q.reshape(p.n_rows, -1).astype(np.float32), act)
    m = np.zeros((p.c.n_pages, 2, 64))
    if score == "one":
        m[:, :, 0] = -7
        m[p.table[0, 5]] = m[p.table[1, 5]] = m[p.table[2, 5]] = -0.5
    elif score > 0:
        m[:, :, 0], m[:, :, 1] = 2, -2.0 ** -24
    else:
        m[:, :, 0] = score
    p.mean = ref.to_bits(m.astype(np.float32), act)
    for n_sel, first, last in ((1, 0, 1), (3, 1, 2), (16, 4, 12), (20, 0, 20), (4, 1, 2)):
        p.check(n_sel, first, last)


@kinds
@pytest.mark.parametrize("n_sel", [4, 70, 300, 512])
def test_own_block_behind_a_list_s_end(dev, act, kv, n_sel):
    """Entries behind a list's end that name the own block again, beside the end, 64 and 256 entries away and in every place: the
    positions behind the row's own stay out.  They hold NaN, or keys of later rows."""
    t = Setup(35, 4, 2, 64, 16, act, kv, [1] * 6 + [9], [150, 145, 159, 145, 9, 97, 157])
    sel = np.full((t.n_rows, 2, n_sel), -1, np.int64)
    for r, s, pos in rows_of(t):
        own = pos // 16
        for h in range(2):
            sel[r, h, :2] = [0, own] if own and (r + h) % 4 else [own, -1]
            end = 2 if own and (r + h) % 4 else 1
            for at in {0: [end + 1], 1: range(end + 1, n_sel, 2), 2: [n_sel - 1], 3: range(end, n_sel), 4: [end + 63],
                       5: [end + 255], 6: [end + 1, n_sel - 1]}[(r + 2 * h) % 7]:
                sel[r, h, min(at, n_sel - 1)] = own
    check(t, n_sel, sel)


@kinds
def test_a_list_repeated(dev, act, kv):
    """Short lists repeated to fill n_sel end where they begin again; also of one block, the own one."""
    t = Setup(36, 8, 2, 128, 32, act, kv, [1, 1, 6], [300, 70, 203])
    sel = np.full((t.n_rows, 2, 12), -1, np.int64)
    for r, s, pos in rows_of(t):
        own = pos // 32
        sel[r, 0] = ([own, 0, own] if r % 2 else [own, 1, 0]) * 4
        sel[r, 1] = [0, own] * 6 if own else [0] * 12
    check(t, 12, sel)
