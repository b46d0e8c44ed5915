"""Arguments that x100_sparse.h refuses, on the host alone, and its sizes."""
import pytest

import x100hip as x
from test_paged_args import A, BAD_BATCH, BAD_CFG, batch, cfg, refused

LD = 1024


def pick(n_sel=4, n_first=1, n_last=1):
    return x.KvSel(n_sel, n_first, n_last)


def means(c=None, b=None, k=A, m=A):
    refused(x.kv_means, c or cfg(), b or batch(), k, m)


def select(c=None, b=None, p=None, q=A, ldq=LD, m=A, s=A):
    refused(x.attn_select, c or cfg(), b or batch(), p or pick(), q, ldq, m, s)


def sparse(c=None, b=None, q=A, ldq=LD, k=A, v=2 * A, scale=1.0, sel=A, n_sel=4, out=A, ldo=LD, ws=A, n=1 << 30):
    a = (c or cfg(), b or batch(), q, ldq, k, v, scale, sel, n_sel, out, ldo)
    refused(x.attn_sparse_ws, *a, ws, n)
    if ws == A and n == 1 << 30:
        refused(x.attn_sparse, *a)


@pytest.mark.parametrize("bad", BAD_CFG, ids=str)
def test_bad_configurations(bad):
    c = cfg(**bad)
    assert x.kv_means_bytes(c) == 0 and x.attn_sparse_workspace_bytes(c, batch(), 4) == 0
    means(c)
    select(c, ldq=1 << 20)
    sparse(c, ldq=1 << 20, ldo=1 << 20)


@pytest.mark.parametrize("bad", BAD_BATCH, ids=str)
def test_bad_batches(bad):
    means(b=batch(**bad))
    select(b=batch(**bad))
    sparse(b=batch(**bad))


def test_bad_pointers_and_strides():
    for p in (None, A + 8):
        means(m=p)
        select(m=p)
        select(q=p)
        sparse(q=p)
        sparse(out=p)
    for p in (None, A + 128):
        means(k=p)
        sparse(k=p)
        sparse(v=p)
    for p in (None, A + 2):
        select(s=p)
        sparse(sel=p)
    for ld in (LD - 8, LD + 4, (1 << 40) + 8):
        select(ldq=ld)
        sparse(ldq=ld)
        sparse(ldo=ld)
    for s in (0.0, -1.0, float("nan"), 2e38, float("inf")):
        sparse(scale=s)
    sparse(v=A)


def test_bad_lists():
    for p in (pick(0, 0, 1), pick(513, 0, 1), pick(4, -1, 1), pick(4, 1, 0), pick(4, 3, 2), pick(4, 1 << 30, 4), pick(4, 0, 5),
              pick(4, 2 ** 31 - 1, 2 ** 31 - 1), pick(-1, 0, 1)):
        select(p=p)
    for n in (0, -1, 513):
        sparse(n_sel=n)
        assert x.attn_sparse_workspace_bytes(cfg(), batch(), n) == 0
    # more blocks than the selection looks at
    select(c=cfg(page=16), b=batch(max_kv=16 * 16384 + 1, table_ld=16385))
    # past one launch
    big = batch(n_rows=(1 << 24) - 1)
    select(b=big)
    sparse(b=big)
    means(c=cfg(n_head=64, n_head_kv=64, act_type=x.T_F16), b=big)


def test_workspace():
    c = cfg(n_head=8, n_head_kv=1, kv_type=x.T_BF16)
    one = x.attn_sparse_workspace_bytes(c, batch(n_rows=1), 64)
    assert one >= 8 * 130 * 4 * 32 and one % 256 == 0            # 64 pages of 64 positions: 32 parts of 128
    for b in (batch(n_rows=1, n_seq=9), batch(n_rows=1, max_q=7), batch(n_rows=1, max_kv=128)):
        assert x.attn_sparse_workspace_bytes(c, b, 64) == one    # by n_rows alone
    assert x.attn_sparse_workspace_bytes(c, batch(n_rows=256), 64) == 0
    assert x.attn_sparse_workspace_bytes(c, batch(n_rows=0), 64) == 0
    sparse(c, batch(n_rows=1), n_sel=64, ws=None)
    sparse(c, batch(n_rows=1), n_sel=64, n=one - 1)
    sparse(c, batch(n_rows=1), n_sel=64, ws=A + 128)
    assert x.kv_means_bytes(cfg()) == 4 * 2 * 128 * 2
    # nothing to do is no error, and needs no device
    assert x.kv_means(cfg(), batch(n_rows=0), A, A) == 0
    assert x.attn_select(cfg(), batch(n_seq=0), pick(), A, LD, A, A) == 0
    assert x.attn_sparse(cfg(), batch(n_rows=0), A, LD, A, 2 * A, 1.0, A, 4, A, LD) == 0


def test_means_of_a_full_launch():
    """Blocks of 16 rows: n_rows is rounded up before it meets the launch's limit (262143 rows by 1024 heads)."""
    c = cfg(n_head=1024, n_head_kv=1024, head_dim=64)
    for n in (262129, 262143, 262144):
        means(c, batch(n_rows=n, max_q=n, max_kv=256, table_ld=4))
