"""Batches whose device arrays break the host's bounds (x100_paged.h): what an append stores, where, and what a
read-back and attention give.  tests/test_paged_rows.py walks the same search on the host."""
import numpy as np
import pytest
import torch

import paged_ref as ref
import x100hip as x
from test_paged_gpu import Setup, kinds, projections, stream, TT

pytestmark = pytest.mark.gpu

# q_start, n_rows, cached positions of each sequence (one number: of all)
BREAKS = [
    ([0, 2, 1, 9], 9, 30),                                       # decreasing
    ([0, 2, 5, 10], 9, 30),                                      # past the rows
    ([0, 2, 5, 9], 9, [-1, 33, 20]),                             # lengths outside 0 .. max_kv
    ([-1, 2, 5, 9], 9, 30),
    ([0, 10, 2, 4, 8], 12, 30),                                  # rows behind an accepted sequence that follows a break
    ([0, 9, 2, 5], 9, 30),
    ([0, 10, 2, 6], 10, 30),
    ([0, 4, 6, 9, 13, 14, 20, 18, 19, 20], 20, 32),              # as many positions as the tables hold
    ([3, 1, 7, 2, 12], 12, [32, 5, 32, 1]),
    ([0, 30, 5, 12, 12, 40], 40, 32),
    ([0, 40, 3, 1 << 30, 20, 40], 40, 32),
    ([0] + [1 + (i * 7) % 60 for i in range(70)] + [64], 64, 32),
]


def setup(q_start, n_rows, kv, act, kvt):
    S = len(q_start) - 1
    kv = kv if isinstance(kv, list) else [kv] * S
    s = Setup(50, 4, 2, 64, 16, act, kvt, [0] * S, [32] * S, max_q=n_rows, max_kv=32)
    s.table = np.ascontiguousarray(s.table[:, :2])               # nothing behind max_kv
    s.q_start, s.n_rows, s.kv_lens = np.array(q_start), n_rows, kv
    # every position has a number already, so that a store into any of them shows
    c = s.c
    K, V = (s.g.standard_normal((c.n_pages, 2, 16, 64)).astype(np.float32) for _ in range(2))
    s.kb, s.vb = c.encode(K, V)
    s.upload()
    return s


def accepted(s):
    """(sequence, first row, rows, positions) of those within the bounds."""
    q = [int(v) for v in s.q_start]
    return [(i, a, b - a, L) for i, (a, b, L) in enumerate(zip(q, q[1:], s.kv_lens))
            if 0 <= a < b <= s.n_rows and b - a <= s.max_q and 0 <= L <= s.max_kv]


@kinds
@pytest.mark.parametrize("q_start,n_rows,kv_len", BREAKS, ids=[str(b[0])[:40] for b in BREAKS])
def test_append_and_read_back(dev, act, kv, q_start, n_rows, kv_len):
    """Only positions of accepted sequences change, and only to their rows; outputs are a row's own or left alone."""
    s = setup(q_start, n_rows, kv_len, act, kv)
    c, hd = s.c, 64
    old = c.decode(s.kb, s.vb)
    rows, vals, keep = projections(s.g, n_rows, 4, 2, hd, ref.F32)
    guard = 8
    out = [torch.full((n_rows + guard, w * hd), -7.0, dtype=TT[act], device=dev) for w in (4, 2, 2)]
    x.kv_append(s.cfg, s.batch, x.KvRows(*rows), s.dk.data_ptr(), s.dv.data_ptr(), out[0].data_ptr(), stream())
    x.kv_read(s.cfg, s.batch, s.dk.data_ptr(), s.dv.data_ptr(), out[1].data_ptr(), out[2].data_ptr(), stream())
    torch.cuda.synchronize()
    new = c.decode(s.dk.cpu().numpy(), s.dv.cpu().numpy())
    q_out, k_out, v_out = (t.float().cpu().numpy().astype(np.float64).reshape(n_rows + guard, -1, hd) for t in out)
    as_act = lambda t: ref.from_bits(ref.to_bits(t, act), act)  # noqa: E731

    def cached(t):   # fp32 rows as the cache holds them
        t = np.asarray(t, np.float32)
        return ref.q4_values(*ref.q4_encode(t)) if kv == ref.Q4 else ref.from_bits(ref.to_bits(t, kv), kv)

    for got, was, first in ((new[0], old[0], 4), (new[1], old[1], 6)):
        want = was.copy()
        for i, r0, n, L in accepted(s):
            for j in range(n):
                p = L - n + j
                if p < 0:
                    continue
                at = (s.table[i][p // 16], slice(None), p % 16)
                row = cached(vals[r0 + j, first:first + 2])
                if np.array_equal(got[at], row):
                    want[at] = row
        assert np.array_equal(got, want)
    sound = all(a <= b for a, b in zip(q_start, q_start[1:]))
    for r in range(n_rows + guard):
        mine = [(i, L - n + r - r0) for i, r0, n, L in accepted(s) if r0 <= r < r0 + n]
        left = [(t[r] == -7).all() for t in (q_out, k_out, v_out)]
        assert left[0] == left[1] == left[2]                      # one search, one answer
        if left[0]:
            assert not (sound and mine), r
            continue
        ok = []
        for i, p in mine:
            if p < 0:
                ok.append(not q_out[r].any() and not k_out[r].any() and not v_out[r].any())
                continue
            at = (s.table[i][p // 16], slice(None), p % 16)
            ok.append(np.array_equal(q_out[r], as_act(vals[r, :4])) and np.array_equal(k_out[r], as_act(new[0][at]))
                      and np.array_equal(v_out[r], as_act(new[1][at])))
        assert any(ok), r


@kinds
@pytest.mark.parametrize("q_start,n_rows,kv_len", BREAKS, ids=[str(b[0])[:40] for b in BREAKS])
def test_attention(dev, act, kv, q_start, n_rows, kv_len):
    """An output is that of an accepted sequence that names the row (of one or another, where several do), or left
    alone; where q_start does not decrease, no named row is left."""
    s = setup(q_start, n_rows, kv_len, act, kv)
    dq, q = s.queries()
    out = s.attend(dq, 256, 0.125).float().cpu().numpy().astype(np.float64).reshape(n_rows, 4, 64)
    K, V = s.c.decode(s.kb, s.vb)
    right, named = out == -7, np.zeros(n_rows, bool)
    for i, r0, n, L in accepted(s):
        want = np.zeros((n, 4, 64))
        tol = ref.attend(s.c, K, V, q[r0:r0 + n], [0, n], [L], [s.table[i]], 0.125, want, n_rows, 32)
        right[r0:r0 + n] |= np.abs(out[r0:r0 + n] - want) <= tol
        named[r0:r0 + n] = True
    assert right.all()
    left = (out == -7).all((1, 2))
    assert left[~named].all()
    if all(a <= b for a, b in zip(q_start, q_start[1:])):
        assert not left[named].any()


def broken(seed, n_seq, most, wrong):
    """Lengths of 0 .. most rows, then `wrong` entries anywhere within the rows."""
    g = np.random.default_rng(seed)
    q = np.concatenate([[0], np.cumsum(g.integers(0, most + 1, n_seq))])
    n_rows = int(q[-1]) + 1
    q[g.integers(0, n_seq + 1, wrong)] = g.integers(0, n_rows + 1, wrong)
    return [int(v) for v in q], n_rows, [int(v) for v in g.integers(0, 33, n_seq)]


MANY = [broken(s, n, m, w) for s, n, m, w in ((1, 600, 3, 1), (2, 600, 2, 5), (3, 520, 3, 40), (4, 30, 40, 3), (5, 70, 20, 6))]


@kinds
@pytest.mark.parametrize("case", range(len(MANY)))
def test_many_sequences(dev, act, kv, case):
    """More sequences than the prompt kernel counts, and prompts without the kernel of few rows beside them."""
    test_append_and_read_back(dev, act, kv, *MANY[case])
    test_attention(dev, act, kv, *MANY[case])


@kinds
def test_a_graph_replayed_over_broken_arrays(dev, act, kv):
    """The arrays break between replays and are put right again: sound replays give what they gave."""
    s = setup([0, 40, 41, 60], 60, [32, 7, 32], act, kv)
    rows, vals, keep = projections(s.g, 60, 4, 2, 64, ref.F32)
    outs = [torch.zeros((60, w), dtype=TT[act], device=dev) for w in (256, 256, 128, 128)]
    n = x.attn_paged_workspace_bytes(s.cfg, s.batch)
    ws = torch.empty(max(n, 256), dtype=torch.uint8, device=dev)

    def call():
        q, o, k, v = (t.data_ptr() for t in outs)
        x.kv_append(s.cfg, s.batch, x.KvRows(*rows), s.dk.data_ptr(), s.dv.data_ptr(), q, stream())
        x.attn_paged_ws(s.cfg, s.batch, q, 256, s.dk.data_ptr(), s.dv.data_ptr(), 0.125, o, 256, ws.data_ptr(), n, stream())
        x.kv_read(s.cfg, s.batch, s.dk.data_ptr(), s.dv.data_ptr(), k, v, stream())

    call()
    torch.cuda.synchronize()
    want, pools = [t.clone() for t in outs], [s.dk.clone(), s.dv.clone()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    sound = s.d_qs.clone()
    for bad in ([0, 40, 3, 60], [50, 10, 45, 60], [0, 70, 3, 8], [-5, 40, 1 << 30, 60]):
        s.d_qs.copy_(torch.tensor(bad, dtype=torch.int32))
        graph.replay()
        s.d_qs.copy_(sound)
        s.dk.copy_(pools[0])     # rows stored for accepted sequences, over their cached positions
        s.dv.copy_(pools[1])
        for t in outs:
            t.fill_(-7)
        graph.replay()
        torch.cuda.synchronize()
        for t, w in zip(outs, want):
            assert torch.equal(t.view(torch.int16), w.view(torch.int16))
