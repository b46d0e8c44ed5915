"""Paged KV cache: append, read-back and attention against plain forms in 64 bits (paged_ref.py)."""
import numpy as np
import pytest
import torch

import paged_ref as ref
import x100hip as x

pytestmark = pytest.mark.gpu

TT = {ref.F32: torch.float32, ref.F16: torch.float16, ref.BF16: torch.bfloat16, ref.I32: torch.int32}


def stream():
    return torch.cuda.current_stream().cuda_stream


def dev_i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32).cuda()


class Setup:
    """A cache of normal values and a batch; the tail of every last page, and the pages of no
    sequence, hold NaN bytes (0xff)."""

    def __init__(self, seed, n_head, n_kv, hd, page, act, kv, q_lens, kv_lens, spare=2, tail_rows=0, max_q=None,
                 max_kv=None, peak=1.0):
        g = self.g = np.random.default_rng(seed)
        self.q_lens, self.kv_lens = list(q_lens), list(kv_lens)
        S = len(q_lens)
        self.max_q = max_q or max(1, max(q_lens))
        self.max_kv = max_kv or max(1, max(kv_lens))
        per = -(-self.max_kv // page) + 1
        need = [-(-n // page) for n in kv_lens]
        n_pages = sum(need) + spare
        c = self.c = ref.Cache(n_head, n_kv, hd, page, n_pages, act, kv)
        free = list(g.permutation(n_pages))
        self.table = np.full((S, per), -1, np.int64)
        used = np.zeros((n_pages, page), bool)
        for s in range(S):
            for i in range(need[s]):
                p = free.pop()
                self.table[s, i] = p
                used[p, :min(page, kv_lens[s] - i * page)] = True
        K, V = ((g.standard_normal((n_pages, n_kv, page, hd)) * peak).astype(np.float32) for _ in range(2))
        hole = ~used[:, None, :, None] & np.ones((1, n_kv, 1, hd), bool)
        self.kb, self.vb = c.encode(np.where(hole, np.float32(np.nan), K), np.where(hole, np.float32(np.nan), V))
        self.cfg = x.KvCfg(n_head, n_kv, hd, page, n_pages, act, kv)
        self.q_start = np.concatenate([[0], np.cumsum(q_lens)])
        self.n_rows = int(self.q_start[-1]) + tail_rows
        self.upload()

    def upload(self):
        self.dk, self.dv = (torch.from_numpy(b.copy()).cuda() for b in (self.kb, self.vb))
        assert self.dk.numel() == x.kv_pool_bytes(self.cfg)
        self.d_qs, self.d_kl = dev_i32(self.q_start), dev_i32(self.kv_lens)
        self.d_tab = dev_i32(self.table)
        self.batch = x.KvBatch(len(self.kv_lens), self.n_rows, self.max_q, self.max_kv, self.table.shape[1],
                               self.d_qs.data_ptr(), self.d_kl.data_ptr(), self.d_tab.data_ptr())

    def queries(self, gain=1.0, pad=0):
        c = self.c
        q = (self.g.standard_normal((self.n_rows, c.n_head * c.hd + pad)) * gain).astype(np.float32)
        bits = ref.to_bits(q, c.act)
        d = torch.from_numpy(bits.view(np.int16)).cuda()
        vals = ref.from_bits(bits, c.act)[:, :c.n_head * c.hd].reshape(self.n_rows, c.n_head, c.hd)
        return d, vals

    def attend(self, dq, ldq, scale, ldo=None, ws=True):
        c = self.c
        ldo = ldo or c.n_head * c.hd
        out = torch.full((self.n_rows, ldo), -7.0, dtype=TT[c.act], device="cuda")
        if ws:
            n = x.attn_paged_workspace_bytes(self.cfg, self.batch)
            w = torch.full((max(n, 256),), 255, dtype=torch.uint8, device="cuda")
            x.attn_paged_ws(self.cfg, self.batch, dq.data_ptr(), ldq, self.dk.data_ptr(), self.dv.data_ptr(), scale,
                            out.data_ptr(), ldo, w.data_ptr(), n, stream())
        else:
            x.attn_paged(self.cfg, self.batch, dq.data_ptr(), ldq, self.dk.data_ptr(), self.dv.data_ptr(), scale,
                         out.data_ptr(), ldo, stream())
        torch.cuda.synchronize()
        return out

    def expected(self, q, scale):
        c = self.c
        K, V = c.decode(self.kb, self.vb)
        want = np.full((self.n_rows, c.n_head, c.hd), -7.0)
        tol = ref.attend(c, K, V, q, self.q_start, self.kv_lens, self.table, scale, want, self.max_q, self.max_kv)
        return want, tol

    def check(self, gain=1.0, scale=None, pad=0, ws=True):
        c = self.c
        scale = scale or c.hd ** -0.5
        dq, q = self.queries(gain, pad)
        out = self.attend(dq, c.n_head * c.hd + pad, scale, ws=ws)
        got = out.float().cpu().numpy().astype(np.float64).reshape(self.n_rows, c.n_head, c.hd)
        want, tol = self.expected(q, scale)
        compare(got, want, tol)
        return out, dq


def compare(got, want, tol):
    assert np.array_equal(np.isnan(got), np.isnan(want)), "NaN in %d places, %d wanted" % (np.isnan(got).sum(), np.isnan(want).sum())
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf])
    fin = np.isfinite(want)
    dist = np.abs(got[fin] - want[fin])
    off = dist - tol[fin]
    assert (off <= 0).all(), "off by %.3g, %.3g allowed (%d of %d outside)" % (
        dist[off.argmax()], tol[fin][off.argmax()], (off > 0).sum(), off.size)


KINDS = [(ref.F16, ref.F16), (ref.BF16, ref.BF16), (ref.F16, ref.Q4), (ref.BF16, ref.Q4)]
kinds = pytest.mark.parametrize("act,kv", KINDS, ids=["f16", "bf16", "f16-q4", "bf16-q4"])


# ---- attention --------------------------------------------------------------------------------------
@kinds
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("page", [16, 64])
def test_single_tokens(dev, act, kv, hd, page):
    lens = [1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 300]
    Setup(1, 8, 2, hd, page, act, kv, [1] * len(lens), lens).check()


@kinds
@pytest.mark.parametrize("n_head,n_kv", [(1, 1), (4, 4), (6, 2), (5, 1), (16, 1), (14, 2)])
def test_head_groups(dev, act, kv, n_head, n_kv):
    Setup(2, n_head, n_kv, 128, 32, act, kv, [1, 3, 1, 6], [40, 3, 200, 77]).check()


@kinds
@pytest.mark.parametrize("page", [16, 32, 128, 256])
@pytest.mark.parametrize("hd", [64, 128])
def test_prompts(dev, act, kv, page, hd):
    Setup(3, 4, 2, hd, page, act, kv, [1, 2, 17, 40, 64, 33], [1, 2, 17, 100, 64, 290]).check()


@kinds
@pytest.mark.parametrize("n_head,n_kv", [(8, 1), (3, 3), (10, 2), (16, 1)])
def test_prompts_of_head_groups(dev, act, kv, n_head, n_kv):
    Setup(4, n_head, n_kv, 128, 64, act, kv, [70, 1, 129], [70, 300, 200]).check()


@kinds
def test_long_cache_splits(dev, act, kv):
    for hd, lens in ((128, [3000, 1, 2049]), (64, [5000])):
        s = Setup(5, 4, 1, hd, 64, act, kv, [1] * len(lens), lens)
        assert x.attn_paged_workspace_bytes(s.cfg, s.batch) > 0
        s.check(gain=3.0)
    Setup(6, 8, 1, 128, 64, act, kv, [3, 1], [2500, 700]).check()
    Setup(7, 4, 1, 128, 64, act, kv, [40, 20], [2500, 700]).check()   # rows of several tiles, split


@kinds
def test_empty_rows_and_sequences(dev, act, kv):
    # no cached position; no rows; more rows than positions (the first ones lie before position 0)
    Setup(8, 4, 2, 128, 32, act, kv, [1, 0, 3, 5, 1, 0], [0, 50, 3, 2, 20, 0], tail_rows=4).check()
    Setup(9, 4, 2, 64, 32, act, kv, [40, 30], [7, 0], tail_rows=1).check()
    Setup(10, 16, 1, 128, 32, act, kv, [0, 0], [10, 0], tail_rows=3).check()


@kinds
def test_refused_sequences_and_rows_left_alone(dev, act, kv):
    s = Setup(11, 4, 2, 128, 32, act, kv, [2, 3, 1, 2, 1], [20, 30, 40, 9, 64], tail_rows=2, max_q=4, max_kv=70)
    s.kv_lens[0], s.kv_lens[2] = -1, 71
    s.upload()
    s.check()
    s = Setup(12, 4, 2, 128, 32, act, kv, [2, 5, 1, 2], [20, 30, 40, 9], max_q=4)
    s.check()                                  # more rows than max_q
    for bad in ([0, 2, 1, 8, 10], [-1, 2, 7, 8, 10], [0, 2, 7, 8, 99], [3, 2, 7, 8, 9]):
        s = Setup(13, 4, 2, 128, 32, act, kv, [2, 5, 1, 2], [20, 30, 40, 9])
        s.q_start = np.array(bad)
        s.upload()
        s.check()


@kinds
def test_pages_that_are_none(dev, act, kv):
    s = Setup(14, 8, 2, 128, 16, act, kv, [1, 3, 20, 1], [100, 70, 90, 16])
    s.table[0, 2], s.table[1, 0], s.table[2, 3], s.table[3, 0] = -1, s.c.n_pages, 1 << 30, -(1 << 31)
    s.upload()
    s.check()


@kinds
def test_shared_pages(dev, act, kv):
    s = Setup(15, 8, 2, 128, 32, act, kv, [1, 1, 4], [100, 100, 100])
    s.table[1, :2] = s.table[0, :2]
    s.table[2, :3] = s.table[0, :3]
    s.upload()
    s.check()


@kinds
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_values_that_are_not_finite_in_unseen_positions(dev, act, kv, bad):
    """An infinity or NaN in a row's key or value reaches the rows that attend to it, and no others."""
    for q, L in (([12], [30]), ([40], [40]), ([130], [150])):
        s = Setup(16, 8, 2, 128, 32, act, kv, q, L)
        c = s.c
        K, V = c.decode(s.kb, s.vb)
        p = L[0] - q[0] // 2
        pg, off = s.table[0][p // 32], p % 32
        V[pg, 0, off, 5] = bad
        K[pg, 1, off, 7] = np.nan
        s.kb, s.vb = c.encode(K.astype(np.float32), V.astype(np.float32))
        s.upload()
        dq, qv = s.queries()
        out = s.attend(dq, 8 * 128, 128 ** -0.5).float().cpu().numpy().astype(np.float64).reshape(-1, 8, 128)
        want, tol = s.expected(qv, 128 ** -0.5)
        first = p - (L[0] - q[0])
        assert np.isfinite(want[:first]).all() and not np.isfinite(want[first:, 0, 5]).any()
        compare(out, want, tol)


@kinds
def test_scores_of_great_size(dev, act, kv):
    # weights that are all but one zero, and queries far from 1
    Setup(17, 4, 2, 128, 64, act, kv, [1, 5, 40], [700, 130, 60]).check(gain=60.0)
    Setup(18, 4, 2, 128, 64, act, kv, [1, 5, 40], [700, 130, 60]).check(gain=1e-4, scale=20.0)
    if act == ref.BF16:
        Setup(19, 4, 2, 128, 64, act, kv, [1, 5, 40], [700, 130, 60]).check(gain=1e15, scale=1e-15)
        Setup(20, 4, 2, 128, 64, act, kv, [1, 5, 40], [700, 130, 60]).check(gain=1e-15, scale=1e15)


@kinds
def test_strides_and_the_plain_form(dev, act, kv):
    s = Setup(21, 4, 2, 64, 32, act, kv, [1, 3, 20], [1200, 50, 60])
    s.check(pad=8, ws=False)
    dq, q = s.queries(pad=24)
    out = s.attend(dq, 4 * 64 + 24, 0.125, ldo=4 * 64 + 40)
    want, tol = s.expected(q, 0.125)
    compare(out[:, :256].float().cpu().numpy().astype(np.float64).reshape(s.n_rows, 4, 64), want, tol)
    assert (out[:, 256:] == -7).all()


@kinds
def test_same_bits_every_time_and_on_another_stream(dev, act, kv):
    s = Setup(22, 8, 2, 128, 64, act, kv, [1, 30, 2], [3000, 400, 900])
    dq, _ = s.queries()
    first = s.attend(dq, 1024, 0.1)
    other = torch.cuda.Stream()
    for i in range(4):
        with torch.cuda.stream(other if i % 2 else torch.cuda.current_stream()):
            again = s.attend(dq, 1024, 0.1, ws=i < 2)
        assert torch.equal(first.view(torch.int16), again.view(torch.int16))


@kinds
def test_graph_replays_follow_the_arrays(dev, act, kv):
    """A captured call reads lengths and pages when it is replayed."""
    s = Setup(23, 8, 2, 128, 32, act, kv, [1, 1, 6], [2000, 100, 50], max_kv=2500, max_q=8)
    dq, q = s.queries()
    out = torch.zeros((s.n_rows, 1024), dtype=TT[act], device=dev)
    n = x.attn_paged_workspace_bytes(s.cfg, s.batch)
    ws = torch.empty(max(n, 256), dtype=torch.uint8, device=dev)

    def call():
        x.attn_paged_ws(s.cfg, s.batch, dq.data_ptr(), 1024, s.dk.data_ptr(), s.dv.data_ptr(), 0.1, out.data_ptr(), 1024,
                        ws.data_ptr(), n, stream())

    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for lens in ([2000, 100, 50], [1500, 64, 6], [1999, 1, 50], [32, 99, 0], [2000, 100, 50]):
        s.kv_lens = lens
        s.d_kl.copy_(dev_i32(lens))
        out.fill_(-7)
        ws.fill_(255)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        out.fill_(-7)
        call()
        torch.cuda.synchronize()
        assert torch.equal(got.view(torch.int16), out.view(torch.int16))
        want, tol = s.expected(q, 0.1)
        compare(got.float().cpu().numpy().astype(np.float64).reshape(s.n_rows, 8, 128), want, tol)


def test_cache_past_32_bit_offsets(dev):
    """Pages whose byte offsets pass 2^32 (in 16 bits: a pool of 4.5 GiB, the last pages used)."""
    page, n_kv, hd = 256, 8, 128
    n_pages = (9 << 29) // (page * n_kv * hd * 2)
    cfg = x.KvCfg(8, n_kv, hd, page, n_pages, ref.F16, ref.F16)
    pools = [torch.zeros(x.kv_pool_bytes(cfg), dtype=torch.uint8, device=dev) for _ in range(2)]
    assert pools[0].numel() > 1 << 32
    L = 300
    tab, qs, kl = dev_i32([[n_pages - 1, n_pages - 2]]), dev_i32([0, L]), dev_i32([L])
    b = x.KvBatch(1, L, L, L, 2, qs.data_ptr(), kl.data_ptr(), tab.data_ptr())
    g = torch.Generator(device="cuda").manual_seed(1)
    src = torch.randn(L, 3 * 1024, generator=g, device=dev).half()
    p = src.data_ptr()
    r = x.KvRows(*[x.Rows(ref.F16, p + 2048 * i, 3 * 1024, None, None) for i in range(3)])
    q_out = torch.empty(L, 1024, dtype=torch.float16, device=dev)
    x.kv_append(cfg, b, r, pools[0].data_ptr(), pools[1].data_ptr(), q_out.data_ptr(), stream())
    k, v = (torch.empty(L, 1024, dtype=torch.float16, device=dev) for _ in range(2))
    x.kv_read(cfg, b, pools[0].data_ptr(), pools[1].data_ptr(), k.data_ptr(), v.data_ptr(), stream())
    assert torch.equal(q_out, src[:, :1024]) and torch.equal(k, src[:, 1024:2048]) and torch.equal(v, src[:, 2048:])
    out = torch.empty_like(q_out)
    x.attn_paged(cfg, b, q_out.data_ptr(), 1024, pools[0].data_ptr(), pools[1].data_ptr(), hd ** -0.5, out.data_ptr(), 1024,
                 stream())
    q, k, v = (t.double().view(L, 8, hd).transpose(0, 1) for t in (q_out, k, v))
    z = q @ k.transpose(1, 2).contiguous() * hd ** -0.5
    z = z.masked_fill(torch.ones(L, L, device=dev).triu(1).bool(), float("-inf")).softmax(-1)
    want = (z @ v).transpose(0, 1).reshape(L, 1024)
    # weights and result rounded to fp16 (2^-11 each), scores in fp32
    tol = (2.0 ** -11 * 1.05 + 1e-4) * (z @ v.abs()).transpose(0, 1).reshape(L, 1024) + 2.0 ** -11 * want.abs() + 1e-7
    assert ((out.double() - want).abs() <= tol).all()


@kinds
@pytest.mark.parametrize("hd,page,L", [(64, 16, 9000), (128, 16, 8500), (64, 256, 8449)])
def test_long_tables(dev, act, kv, hd, page, L):
    """Caches whose page list does not fit a block's as a whole, and pages larger than a split's step."""
    Setup(24, 2, 1, hd, page, act, kv, [1, 1], [L, 77]).check()
    s = Setup(25, 4, 1, hd, page, act, kv, [1, 2], [L, 300])
    s.table[0, 3] = -1          # a page that is none, far from the end
    s.upload()
    s.check()


@kinds
@pytest.mark.parametrize("n_head,n_kv,hd", [(2, 2, 128), (3, 1, 64), (16, 1, 128), (7, 1, 128), (2, 1, 64)])
def test_prompts_of_many_tiles(dev, act, kv, n_head, n_kv, hd):
    """Prompts over several blocks of rows and many tiles of positions, with a decode row among them, against
    64-bit products on the GPU."""
    q, L = [300, 1, 33, 700], [300, 1500, 1700, 777]
    s = Setup(26, n_head, n_kv, hd, 32, act, kv, q, L)
    dq, qv = s.queries(gain=1.5)
    out = s.attend(dq, n_head * hd, hd ** -0.5).double().view(s.n_rows, n_head, hd)
    K, V = (torch.from_numpy(np.nan_to_num(t)).cuda() for t in s.c.decode(s.kb, s.vb))
    Q = torch.from_numpy(qv).cuda()
    u = ref.HALF_STEP[act] + ref.HALF_STEP[ref.F16 if kv == ref.Q4 else act]
    for i in range(len(q)):
        pg = torch.from_numpy(s.table[i][:-(-L[i] // 32)]).cuda()
        k, v = (t[pg].transpose(0, 1).reshape(n_kv, -1, hd)[:, :L[i]] for t in (K, V))
        r0, n = int(s.q_start[i]), q[i]
        hidden = torch.arange(L[i], device=dev)[None] > torch.arange(L[i] - n, L[i], device=dev)[:, None]
        for h in range(n_head):
            kk, vv = k[h * n_kv // n_head].contiguous(), v[h * n_kv // n_head].contiguous()
            z = (Q[r0:r0 + n, h] @ kk.T.contiguous() * hd ** -0.5).masked_fill(hidden, float("-inf")).softmax(-1)
            want, size = z @ vv, z @ vv.abs()
            # the weights' and the result's 16-bit rounding; the scores in fp32
            assert ((out[r0:r0 + n, h] - want).abs() <= (1.01 * u + 1e-4) * size + 1e-6).all(), (i, h)


@kinds
@pytest.mark.parametrize("n_head,n_kv,q,L", [
    (8, 1, [1, 300, 1, 4, 5, 1, 1, 1, 1], [3000, 700, 1, 900, 2000, 17, 0, 256, 4000]),    # 8 .. 40 rows beside a prompt
    (2, 2, [32, 33, 1, 16, 17, 500, 1, 1, 1, 1, 1, 1, 1, 1, 1], [50, 2000, 1500, 16, 900, 500] + [9] * 9),
    (4, 2, [0, 0, 257, 0, 1, 0, 0, 0], [0, 5, 1300, 9, 1300, 1, 1, 1]),                   # sequences without rows
    (16, 1, [2, 70, 1, 3] + [1] * 6, [2500] * 10),
])
def test_prompts_beside_single_tokens(dev, act, kv, n_head, n_kv, q, L):
    """Batches in which sequences of few rows and of many take different kernels, each with its splits."""
    for hd, page in ((64, 16), (128, 64)):
        Setup(28, n_head, n_kv, hd, page, act, kv, q, L).check()


@kinds
@pytest.mark.parametrize("n_seq", [65, 130, 512, 513, 700])
def test_prompts_of_many_sequences(dev, act, kv, n_seq):
    """More sequences than a wave counts at a time, and than are counted at all."""
    g = np.random.default_rng(n_seq)
    q = [int(n) for n in g.integers(33, 40, n_seq)]     # every one long
    Setup(30, 2, 1, 64, 16, act, kv, q, [n + int(e) for n, e in zip(q, g.integers(0, 30, n_seq))]).check()
    q = [1] * n_seq                                     # a few long among single tokens
    q[0], q[n_seq // 2], q[-1] = 40, 300, 150
    Setup(31, 2, 1, 64, 16, act, kv, q, [n + int(e) for n, e in zip(q, g.integers(0, 30, n_seq))]).check()


@kinds
@pytest.mark.parametrize("n_head,q", [(2, 16), (8, 4), (8, 8), (16, 3), (16, 1)])
def test_tiles_of_few_rows(dev, act, kv, n_head, q):
    """Two to four tiles of rows per sequence, whole and ragged, with few splits and many."""
    for n_seq, L in ((1, 5000), (3, 1100), (40, 70)):
        Setup(32, n_head, 1, 64, 16, act, kv, [q] * n_seq, [L - 7 * i % 50 for i in range(n_seq)]).check()
        Setup(33, n_head, 1, 64, 16, act, kv, [q] + [1] * (n_seq - 1), [L - i for i in range(n_seq)]).check()


@kinds
def test_rows_of_a_wider_bound(dev, act, kv):
    """The launch sized for more rows and positions than a sequence has (as a captured one is)."""
    for q, L in (([1, 2, 1], [700, 40, 2000]), ([60, 1, 5], [900, 1, 2000]), ([130, 100, 90], [130, 400, 1000])):
        Setup(29, 4, 2, 64, 16, act, kv, q, L, max_q=2000, max_kv=5000).check()


def test_batches_past_one_launch(dev):
    """Refused by their bounds alone, before anything is enqueued (the arrays are never read)."""
    some = torch.zeros(4096, dtype=torch.int32, device=dev)
    pools = [torch.zeros(256, dtype=torch.uint8, device=dev) for _ in range(2)]
    p = some.data_ptr()
    c = x.KvCfg(1024, 1024, 64, 16, 1, ref.F16, ref.F16)
    b = x.KvBatch(65535, (1 << 24) - 1, 1000, 16, 1, p, p, p)
    with pytest.raises(x.X100Error):
        x.attn_paged(c, b, p, 65536, pools[0].data_ptr(), pools[1].data_ptr(), 1.0, p, 65536, stream())
    assert x.attn_paged_workspace_bytes(c, b) == 0
    rows = [x.Rows(ref.F16, p, 65536, None, None) for _ in range(3)]
    with pytest.raises(x.X100Error):
        x.kv_append(c, b, x.KvRows(*rows, None, None, 0.0, None, 0), pools[0].data_ptr(), pools[1].data_ptr(), p, stream())
    torch.cuda.synchronize()
    assert not some.any()


@kinds
def test_two_calls_at_once(dev, act, kv):
    """Calls on two streams at the same time, each with its own workspace (and through the library's)."""
    sets = [Setup(27 + i, 8, 2, 128, 64, act, kv, [1, q], [3000, 500]) for i, q in enumerate((1, 60))]
    dqs = [s.queries()[0] for s in sets]
    alone = [s.attend(d, 1024, 0.1) for s, d in zip(sets, dqs)]
    streams = [torch.cuda.Stream() for _ in sets]
    for ws in (True, False):
        outs, keep = [], []
        torch.cuda.synchronize()
        for s, d, st in zip(sets, dqs, streams):
            out = torch.zeros_like(alone[len(outs)])
            n = x.attn_paged_workspace_bytes(s.cfg, s.batch)
            w = torch.empty(max(n, 256), dtype=torch.uint8, device=dev)
            torch.cuda.synchronize()
            for _ in range(20):
                args = (s.cfg, s.batch, d.data_ptr(), 1024, s.dk.data_ptr(), s.dv.data_ptr(), 0.1, out.data_ptr(), 1024)
                if ws:
                    x.attn_paged_ws(*args, w.data_ptr(), n, st.cuda_stream)
                else:
                    x.attn_paged(*args, st.cuda_stream)
            outs.append(out)
            keep.append(w)
        torch.cuda.synchronize()
        for a, b in zip(alone, outs):
            assert torch.equal(a.view(torch.int16), b.view(torch.int16))


@kinds
def test_a_decode_step_in_a_graph(dev, act, kv):
    """Append, attention and read-back captured once and replayed as the sequences grow, with eager calls
    between the replays."""
    n_seq, page, max_kv = 3, 16, 80
    c = x.KvCfg(4, 2, 64, page, 20, act, kv)
    pools = [[torch.zeros(x.kv_pool_bytes(c), dtype=torch.uint8, device=dev) for _ in range(2)] for _ in range(2)]
    g = np.random.default_rng(5)
    tab = dev_i32(g.permutation(20)[:15].reshape(3, 5))
    qs, kl = dev_i32([0, 1, 2, 3]), dev_i32([1, 1, 1])
    b = x.KvBatch(n_seq, n_seq, 1, max_kv, 5, qs.data_ptr(), kl.data_ptr(), tab.data_ptr())
    rows, vals, keep = projections(g, n_seq, 4, 2, 64, ref.F32)
    rope = torch.empty(max_kv * 64, device=dev)
    x.rope_table(64, max_kv, 1e4, rope.data_ptr(), stream())
    r = x.KvRows(*rows, None, None, 0.0, rope.data_ptr(), max_kv)
    bufs = [[torch.zeros(n_seq, w, dtype=TT[act], device=dev) for w in (256, 256, 128, 128)] for _ in range(2)]
    ws = torch.empty(max(256, x.attn_paged_workspace_bytes(c, b)), dtype=torch.uint8, device=dev)

    def step(i):
        (q, o, k, v), (kp, vp) = bufs[i], pools[i]
        x.kv_append(c, b, r, kp.data_ptr(), vp.data_ptr(), q.data_ptr(), stream())
        x.attn_paged_ws(c, b, q.data_ptr(), 256, kp.data_ptr(), vp.data_ptr(), 0.125, o.data_ptr(), 256, ws.data_ptr(),
                        ws.numel(), stream())
        x.kv_read(c, b, kp.data_ptr(), vp.data_ptr(), k.data_ptr(), v.data_ptr(), stream())

    step(0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(0)
    for p in pools:
        for t in p:
            t.zero_()
    for n in range(1, 40):
        kl.copy_(dev_i32([n, 2 * n, n // 2]))
        keep[-1].normal_()          # the step's projections
        graph.replay()
        torch.cuda.synchronize()
        step(1)
        torch.cuda.synchronize()
        for s, t in zip(bufs[0] + pools[0], bufs[1] + pools[1]):
            assert torch.equal(s.view(torch.uint8), t.view(torch.uint8)), n


# ---- append and read --------------------------------------------------------------------------------
def projections(g, n, n_head, n_kv, hd, t, split=False):
    """Rows of q | k | v of one type: (KvRows' three Rows, fp32 values [n][heads][hd], keep)."""
    W = (n_head + 2 * n_kv) * hd
    widths = [n_head * hd, n_kv * hd, n_kv * hd]
    if t == ref.I32:
        a = torch.from_numpy(g.integers(-60000, 60000, (n, W)).astype(np.int32))
        rs = torch.from_numpy((g.random(n) * 1e-2 + 1e-3).astype(np.float32))
        cs = torch.from_numpy((g.random(W) * 1e-2 + 1e-3).astype(np.float32))
        vals = (a.float() * rs[:, None]) * cs
    else:
        a = torch.from_numpy((g.standard_normal((n, W)) * 2).astype(np.float32)).to(TT[t])
        rs = cs = None
        vals = a.float()
    keep = [s.cuda() for s in (rs, cs) if s is not None]
    out, col = [], 0
    whole = a.cuda()
    for w in widths:
        if split:    # matrices of their own
            part = a[:, col:col + w].contiguous().cuda()
            keep.append(part)
            ptr, ld = part.data_ptr(), w
        else:
            ptr, ld = whole.data_ptr() + col * a.element_size(), W
        out.append(x.Rows(t, ptr, ld, keep[0].data_ptr() if rs is not None else None,
                          keep[1].data_ptr() + 4 * col if rs is not None else None))
        col += w
    return out, vals.numpy().reshape(n, -1, hd), keep + [whole]


def append_case(seed, n_head, n_kv, hd, page, act, kv, st, q_lens, kv_lens, norm, rope, tail=0, bad_page=None, split=False,
                max_q=None):
    s = Setup(seed, n_head, n_kv, hd, page, act, kv, q_lens, kv_lens, tail_rows=tail, max_q=max_q)
    c = s.c
    # the cached part of a sequence has numbers, its new positions (and the rest) 0xff bytes: a store
    # that touches a neighbour shows
    before = c.decode(s.kb, s.vb)
    if bad_page:
        s.table[bad_page[0], bad_page[1]] = bad_page[2]
        s.upload()
    rows, vals, keep = projections(s.g, s.n_rows, n_head, n_kv, hd, st, split)
    qn, kn = ((1 + 0.3 * s.g.standard_normal(hd)).astype(np.float32) for _ in range(2))
    dqn, dkn = torch.from_numpy(qn).cuda(), torch.from_numpy(kn).cuda()
    table = torch.empty(s.max_kv * hd, device="cuda")
    x.rope_table(hd, s.max_kv, 1e4, table.data_ptr(), stream())
    r = x.KvRows(*rows, dqn.data_ptr() if norm else None, dkn.data_ptr() if norm else None, 1e-6,
                 table.data_ptr() if rope else None, s.max_kv)
    q_out = torch.full((s.n_rows, n_head * hd), -7.0, dtype=TT[act], device="cuda")
    x.kv_append(s.cfg, s.batch, r, s.dk.data_ptr(), s.dv.data_ptr(), q_out.data_ptr(), stream())
    k_out = torch.full((s.n_rows, n_kv * hd), -7.0, dtype=TT[act], device="cuda")
    v_out = torch.full_like(k_out, -7.0)
    x.kv_read(s.cfg, s.batch, s.dk.data_ptr(), s.dv.data_ptr(), k_out.data_ptr(), v_out.data_ptr(), stream())
    torch.cuda.synchronize()
    K, V = c.decode(s.dk.cpu().numpy(), s.dv.cpu().numpy())
    f64 = lambda t: t.float().cpu().numpy().astype(np.float64).reshape(s.n_rows, -1, hd)  # noqa: E731
    q_out, k_out, v_out = f64(q_out), f64(k_out), f64(v_out)
    u = ref.HALF_STEP[act]
    tiny = 2.0 ** -25 if act == ref.F16 else 1e-38
    touched = np.zeros((c.n_pages, page), bool)
    exact_k = not norm and not rope
    for i in range(len(q_lens)):
        q0, n, L = int(s.q_start[i]), q_lens[i], kv_lens[i]
        for j in range(n):
            row, pos = q0 + j, L - n + j
            if n > s.max_q:
                assert (q_out[row] == -7).all() and (k_out[row] == -7).all() and (v_out[row] == -7).all()
                continue
            if pos < 0:
                assert not q_out[row].any() and not k_out[row].any() and not v_out[row].any()
                continue
            t = vals[row].astype(np.float64)
            q, k, v = t[:n_head], t[n_head:n_head + n_kv], t[n_head + n_kv:]
            if norm:
                q, k = ref.head_norm(q, qn.astype(np.float64), 1e-6), ref.head_norm(k, kn.astype(np.float64), 1e-6)
            mag = lambda z: np.sqrt(z[..., :hd // 2] ** 2 + z[..., hd // 2:] ** 2).repeat(2, 0).reshape(z.shape[0], 2, -1).reshape(z.shape)  # noqa: E731
            # fp32 steps: the mean of hd squares, root, quotient, two products, and the rotation's table
            # entry, product and sum (of the pair's size)
            eq, ek = ((hd / 2 + 12) * 2.0 ** -24 * mag(z) if norm else 4 * 2.0 ** -24 * mag(z) for z in (q, k))
            if rope:
                q, k = ref.rotate(q, pos, 1e4), ref.rotate(k, pos, 1e4)
            else:
                eq, ek = ((hd / 2 + 12) * 2.0 ** -24 * np.abs(z) * norm for z in (q, k))
            assert (np.abs(q_out[row] - q) <= u * np.abs(q) + (1 + u) * eq + tiny).all()
            pg = s.table[i][pos // page]
            if not 0 <= pg < c.n_pages:
                assert not k_out[row].any() and not v_out[row].any()
                continue
            off = pos % page
            touched[pg, off] = True
            gk, gv = K[pg, :, off], V[pg, :, off]
            # what is read back is what the cache holds, rounded to act
            assert np.array_equal(k_out[row], ref.from_bits(ref.to_bits(gk, act), act))
            assert np.array_equal(v_out[row], ref.from_bits(ref.to_bits(gv, act), act))
            if kv == ref.Q4:
                assert np.array_equal(gv, ref.q4_values(*ref.q4_encode(v.astype(np.float32))))
                if exact_k:
                    assert np.array_equal(gk, ref.q4_values(*ref.q4_encode(k.astype(np.float32))))
                else:
                    z = k.reshape(-1, 32)
                    st_ = ((z.max(1) - z.min(1)) / 15)[:, None]
                    e = ek.reshape(-1, 32)
                    # half a step; the step's and the minimum's fp16 rounding; the value's; and fp32's
                    bound = st_ * (0.5 + 16 * 2.0 ** -11) + 3 * 2.0 ** -11 * np.abs(z).max(1)[:, None] + 4 * e.max(1)[:, None]
                    assert (np.abs(gk.reshape(-1, 32) - z) <= bound).all()
            else:
                assert np.array_equal(gv, ref.from_bits(ref.to_bits(v.astype(np.float32), act), act))
                assert (np.abs(gk - k) <= u * np.abs(k) + (1 + u) * ek + tiny).all()
    assert (q_out[int(s.q_start[-1]):] == -7).all() and (k_out[int(s.q_start[-1]):] == -7).all()
    # every other position holds what it held
    keep_mask = ~touched
    for got, old in ((K, before[0]), (V, before[1])):
        a, b = got.transpose(0, 2, 1, 3)[keep_mask], old.transpose(0, 2, 1, 3)[keep_mask]
        assert np.array_equal(a, b, equal_nan=True)


@kinds
@pytest.mark.parametrize("st", [ref.F32, ref.F16, ref.BF16, ref.I32], ids=["f32", "f16", "bf16", "i32"])
@pytest.mark.parametrize("hd", [64, 128])
def test_append(dev, act, kv, st, hd):
    append_case(1, 4, 2, hd, 32, act, kv, st, [1, 9, 1, 30, 8, 16], [40, 9, 8, 50, 24, 33], True, True)
    append_case(2, 3, 3, hd, 16, act, kv, st, [1, 2, 3, 17], [1, 9, 70, 17], False, False, split=True)
    append_case(3, 2, 1, hd, 64, act, kv, st, [5, 1], [70, 64], False, True)
    append_case(4, 5, 1, hd, 256, act, kv, st, [1, 4], [13, 300], True, False)


@kinds
@pytest.mark.parametrize("st", [ref.F32, ref.I32], ids=["f32", "i32"])
def test_append_many_groups(dev, act, kv, st):
    """Enough values for a scale or a number that is rounded once too often, or not from fp32, to show."""
    append_case(40, 8, 8, 128, 64, act, kv, st, [3000], [3000], False, False)


@kinds
def test_append_odd_batches(dev, act, kv):
    # empty sequences, rows before position 0, rows behind the last sequence
    append_case(5, 4, 2, 128, 16, act, kv, ref.F32, [0, 3, 5, 0, 12, 1, 0], [10, 3, 2, 0, 7, 0, 5], True, True, tail=5)
    # pages that are none; a sequence with more rows than max_q
    append_case(6, 4, 2, 64, 16, act, kv, ref.BF16, [20, 2], [40, 20], True, True, bad_page=(0, 1, 1 << 30))
    append_case(7, 4, 2, 64, 16, act, kv, ref.BF16, [20, 2], [40, 20], True, True, bad_page=(0, 2, -1))
    append_case(8, 4, 2, 64, 16, act, kv, ref.BF16, [3, 9, 1], [40, 20, 17], True, True, max_q=4, tail=1)


@kinds
@pytest.mark.parametrize("n_seq", [63, 64, 65, 200, 4500])
def test_append_many_sequences(dev, act, kv, n_seq):
    g = np.random.default_rng(n_seq)
    q = g.integers(0, 3, n_seq)
    append_case(9, 1, 1, 64, 16, act, kv, ref.F16, q.tolist(), (q + g.integers(0, 20, n_seq)).tolist(), False, False, tail=2)


@kinds
def test_append_refused_sequences(dev, act, kv):
    s = Setup(30, 4, 2, 128, 16, act, kv, [2, 3, 4], [20, 30, 9])
    rows, vals, keep = projections(s.g, s.n_rows, 4, 2, 128, ref.F32)
    r = x.KvRows(*rows)
    for qs, kl in (([0, 2, 1, 9], [20, 30, 9]), ([0, 2, 5, 10], [20, 30, 9]), ([0, 2, 5, 9], [-1, 31, 31]),
                   ([-1, 2, 5, 9], [20, 31, 31])):
        s.q_start, s.kv_lens = np.array(qs), kl
        s.upload()
        q_out = torch.full((s.n_rows, 512), -7.0, dtype=TT[act], device=dev)
        x.kv_append(s.cfg, s.batch, r, s.dk.data_ptr(), s.dv.data_ptr(), q_out.data_ptr(), stream())
        torch.cuda.synchronize()
        ok = [0 <= a <= b <= s.n_rows and b - a <= s.max_q and 0 <= n <= s.max_kv for a, b, n in zip(qs, qs[1:], kl)]
        for i, fine in enumerate(ok):
            if not fine:
                lo, hi = max(0, qs[i]), min(s.n_rows, qs[i + 1])
                other = [j for j in range(len(ok)) if ok[j] and qs[j] < hi and qs[j + 1] > lo]
                if not other:
                    assert (q_out[lo:hi] == -7).all()


@kinds
def test_append_groups_that_are_not_finite(dev, act, kv):
    if kv != ref.Q4:
        return
    s = Setup(31, 1, 1, 64, 16, act, kv, [4], [4])
    t = s.g.standard_normal((4, 3, 64)).astype(np.float32)
    t[0, 1:, 3], t[1, 1:, 40], t[2, 1:, 0], t[3, 1:, 63] = np.inf, np.nan, 1e6, -1e6
    d = torch.from_numpy(t.reshape(4, 192)).cuda()
    r = x.KvRows(*[x.Rows(ref.F32, d.data_ptr() + 256 * i, 192, None, None) for i in range(3)])
    q_out = torch.empty((4, 64), dtype=TT[act], device=dev)
    x.kv_append(s.cfg, s.batch, r, s.dk.data_ptr(), s.dv.data_ptr(), q_out.data_ptr(), stream())
    torch.cuda.synchronize()
    K, V = s.c.decode(s.dk.cpu().numpy(), s.dv.cpu().numpy())
    for got, i in ((K, 1), (V, 2)):
        for p in range(4):
            want = ref.q4_values(*ref.q4_encode(t[p, i]))
            assert np.array_equal(got[s.table[0, 0], 0, p], want, equal_nan=True) and np.isnan(want).sum() == 32


@kinds
def test_append_keys_and_values_only(dev, act, kv):
    s = Setup(32, 4, 2, 128, 16, act, kv, [3, 1], [20, 30])
    rows, vals, keep = projections(s.g, s.n_rows, 4, 2, 128, ref.F32)
    r = x.KvRows(x.Rows(0, None, 0, None, None), rows[1], rows[2])
    x.kv_append(s.cfg, s.batch, r, s.dk.data_ptr(), s.dv.data_ptr(), None, stream())
    both = [s.dk.clone(), s.dv.clone()]
    s.upload()
    q_out = torch.empty((4, 512), dtype=TT[act], device=dev)
    x.kv_append(s.cfg, s.batch, x.KvRows(*rows), s.dk.data_ptr(), s.dv.data_ptr(), q_out.data_ptr(), stream())
    assert torch.equal(both[0], s.dk) and torch.equal(both[1], s.dv)


@pytest.mark.parametrize("hd,base", [(64, 1e4), (128, 1e6)])
def test_rope_table(dev, hd, base):
    n = 50001
    t = torch.empty(n, hd // 2, 2, device=dev)
    x.rope_table(hd, n, base, t.data_ptr(), stream())
    a = np.arange(n)[:, None] * float(np.float32(base)) ** (-np.arange(0, hd, 2) / hd)
    got = t.cpu().numpy().astype(np.float64)
    # one rounding, and the angle's own error in 64 bits (pow within a few ulp, times 50000)
    assert np.abs(got[..., 0] - np.cos(a)).max() <= 2.0 ** -24 + 50000 * 8 * 2.0 ** -53
    assert np.abs(got[..., 1] - np.sin(a)).max() <= 2.0 ** -24 + 50000 * 8 * 2.0 ** -53


# ---- the operators together ---------------------------------------------------------------------------
@kinds
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_half_of_a_layer(dev, act, kv, hd):
    """A batch's attention half on int8 weights: norm to int8, Wq|Wk|Wv by the int8 GEMM, its int32
    sums appended (norms, rotation), attention, the output to int8, Wo, and the next norm with the
    residual.  First a prompt, then single tokens behind it; against 64 bits at every stage, each from
    the stage's own input."""
    n_head, n_kv, d, page, S = 8, 2, 512, 32, 3
    g = np.random.default_rng(77)
    W = (n_head + 2 * n_kv) * hd
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()  # noqa: E731
    wqkv, wo = t(g.integers(-127, 128, (d, W)).astype(np.int8)), t(g.integers(-127, 128, (n_head * hd, d)).astype(np.int8))
    s_qkv, s_o = (t((g.random(n) * 1e-4 + 5e-4).astype(np.float32)) for n in (W, d))
    n1, n2 = (t((1 + 0.2 * g.standard_normal(d)).astype(np.float32)) for _ in range(2))
    qn, kn = (t((1 + 0.2 * g.standard_normal(hd)).astype(np.float32)) for _ in range(2))
    lens = [37, 1, 64]
    max_kv = 70
    per = -(-max_kv // page)
    table = g.permutation(S * per).reshape(S, per)
    c = ref.Cache(n_head, n_kv, hd, page, S * per, act, kv)
    cfg = x.KvCfg(n_head, n_kv, hd, page, S * per, act, kv)
    pools = [torch.full((x.kv_pool_bytes(cfg),), 255, dtype=torch.uint8, device=dev) for _ in range(2)]
    rope = torch.empty(max_kv * hd, device=dev)
    x.rope_table(hd, max_kv, 1e6, rope.data_ptr(), stream())
    d_tab = dev_i32(table)
    cached = [0] * S
    for q_lens in (lens, [1] * S, [2, 1, 3]):
        n = sum(q_lens)
        cached = [a + b for a, b in zip(cached, q_lens)]
        qs = np.concatenate([[0], np.cumsum(q_lens)])
        d_qs, d_kl = dev_i32(qs), dev_i32(cached)
        b = x.KvBatch(S, n, max(q_lens), max_kv, per, d_qs.data_ptr(), d_kl.data_ptr(), d_tab.data_ptr())
        h = t(g.standard_normal((n, d)).astype(np.float32))
        h0 = h.clone()
        q8, sc = torch.empty((n, d), dtype=torch.int8, device=dev), torch.empty(n, device=dev)
        x.add_rmsnorm_i8(n, d, x.Rows(ref.F32, h.data_ptr(), d, None, None), None, n1.data_ptr(), 1e-6, None, 0,
                         q8.data_ptr(), sc.data_ptr(), stream())
        c32 = torch.empty((n, W), dtype=torch.int32, device=dev)
        x.gemm_dev_set(n, W, d, q8.data_ptr(), wqkv.data_ptr(), c32.data_ptr(), stream())
        part = lambda col: x.Rows(ref.I32, c32.data_ptr() + 4 * col, W, sc.data_ptr(), s_qkv.data_ptr() + 4 * col)  # noqa: E731
        r = x.KvRows(part(0), part(n_head * hd), part((n_head + n_kv) * hd), qn.data_ptr(), kn.data_ptr(), 1e-6,
                     rope.data_ptr(), max_kv)
        q_out = torch.empty((n, n_head * hd), dtype=TT[act], device=dev)
        x.kv_append(cfg, b, r, pools[0].data_ptr(), pools[1].data_ptr(), q_out.data_ptr(), stream())
        att = torch.empty_like(q_out)
        x.attn_paged(cfg, b, q_out.data_ptr(), n_head * hd, pools[0].data_ptr(), pools[1].data_ptr(), hd ** -0.5,
                     att.data_ptr(), n_head * hd, stream())
        a8, asc = torch.empty((n, n_head * hd), dtype=torch.int8, device=dev), torch.empty(n, device=dev)
        x.quant_i8(n, n_head * hd, x.Rows(act, att.data_ptr(), n_head * hd, None, None), a8.data_ptr(), asc.data_ptr(),
                   stream())
        o32 = torch.empty((n, d), dtype=torch.int32, device=dev)
        x.gemm_dev_set(n, d, n_head * hd, a8.data_ptr(), wo.data_ptr(), o32.data_ptr(), stream())
        h8, hsc = torch.empty((n, d), dtype=torch.int8, device=dev), torch.empty(n, device=dev)
        x.add_rmsnorm_i8(n, d, x.Rows(ref.F32, h.data_ptr(), d, None, None),
                         x.Rows(ref.I32, o32.data_ptr(), d, asc.data_ptr(), s_o.data_ptr()), n2.data_ptr(), 1e-6,
                         h.data_ptr(), d, h8.data_ptr(), hsc.data_ptr(), stream())
        torch.cuda.synchronize()
        # every stage from its own input
        hn = h0.cpu().numpy() * n1.cpu().numpy()
        assert np.array_equal(q8.cpu().numpy(), ref.codes_f32(hn)[0])
        assert torch.equal(c32.cpu(), (q8.cpu().double() @ wqkv.cpu().double()).to(torch.int32))
        real = c32.cpu().numpy().astype(np.float64) * np.outer(sc.cpu().numpy(), s_qkv.cpu().numpy().astype(np.float64))
        qkv = real.reshape(n, -1, hd)
        K, V = c.decode(pools[0].cpu().numpy(), pools[1].cpu().numpy())
        f64 = lambda z: z.float().cpu().numpy().astype(np.float64).reshape(n, n_head, hd)  # noqa: E731
        for i in range(S):
            for j in range(q_lens[i]):
                pos, row = cached[i] - q_lens[i] + j, int(qs[i]) + j
                q = ref.rotate(ref.head_norm(qkv[row, :n_head], qn.cpu().numpy().astype(np.float64), 1e-6), pos, 1e6)
                u = ref.HALF_STEP[act]
                size = np.abs(q).max(-1, keepdims=True) * 1.5
                assert (np.abs(f64(q_out)[row] - q) <= u * np.abs(q) + (hd / 2 + 16) * 2.0 ** -24 * size + 2.0 ** -25).all()
                k = ref.rotate(ref.head_norm(qkv[row, n_head:n_head + n_kv], kn.cpu().numpy().astype(np.float64), 1e-6), pos, 1e6)
                gk = K[table[i][pos // page], :, pos % page]
                step = 2.0 ** -8 * np.abs(k) if kv != ref.Q4 else (k.max() - k.min()) / 15 * 0.52 + 2.0 ** -9 * np.abs(k).max()
                assert (np.abs(gk - k) <= step + 1e-4).all()
        want = np.zeros((n, n_head, hd))
        tol = ref.attend(c, K, V, f64(q_out), qs, cached, table, hd ** -0.5, want, max(q_lens), max_kv)
        compare(f64(att), want, tol)
        assert np.array_equal(a8.cpu().numpy(), ref.codes_f32(att.float().cpu().numpy())[0])
        assert torch.equal(o32.cpu(), (a8.cpu().double() @ wo.cpu().double()).to(torch.int32))
        o = (o32.cpu().float() * asc.cpu()[:, None]) * s_o.cpu()
        assert torch.equal(h.cpu(), h0.cpu() + o)
        assert np.array_equal(h8.cpu().numpy(), ref.codes_f32(h.cpu().numpy() * n2.cpu().numpy())[0])
