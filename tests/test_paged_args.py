"""Refusals of x100_rows.h / x100_paged.h (no GPU: an argument error returns before the device is
looked at) and the plain forms' own round trips."""
import ctypes

import numpy as np
import pytest

import paged_ref as ref
import x100hip as x

A = 1 << 20   # a 256-byte aligned address that is never read: every call here is refused


def cfg(**k):
    d = dict(n_head=8, n_head_kv=2, head_dim=128, page=64, n_pages=4, act_type=x.T_BF16, kv_type=x.KV_Q4)
    d.update(k)
    return x.KvCfg(*[d[n] for n, _ in x.KvCfg._fields_])


def batch(**k):
    d = dict(n_seq=2, n_rows=3, max_q=2, max_kv=100, table_ld=2, q_start=A, kv_len=A, block_table=A)
    d.update(k)
    return x.KvBatch(*[d[n] for n, _ in x.KvBatch._fields_])


def rows(t=x.T_F32, p=A, ld=4096, rs=None, cs=None):
    return x.Rows(t, p, ld, rs, cs)


def refused(f, *a):
    with pytest.raises(x.X100Error) as e:
        f(*a)
    assert e.value.code == x.X100_EINVAL


BAD_CFG = [dict(n_head=0), dict(n_head_kv=0), dict(n_head=9), dict(n_head=34), dict(head_dim=96), dict(head_dim=256),
           dict(page=8), dict(page=48), dict(page=512), dict(n_pages=0), dict(act_type=x.T_F32),
           dict(kv_type=x.T_F16), dict(kv_type=5), dict(n_head=2048, n_head_kv=2048)]
BAD_BATCH = [dict(n_seq=-1), dict(n_seq=65536), dict(n_rows=-1), dict(n_rows=1 << 24), dict(max_q=0), dict(max_kv=0),
             dict(table_ld=1), dict(table_ld=0), dict(q_start=None), dict(kv_len=None), dict(block_table=None),
             dict(kv_len=A + 2), dict(max_q=(1 << 20) + 1)]


@pytest.mark.parametrize("bad", BAD_CFG, ids=str)
def test_bad_configurations(bad):
    c, b = cfg(**bad), batch()
    assert x.kv_pool_bytes(c) == 0
    assert x.attn_paged_workspace_bytes(c, b) == 0
    refused(x.attn_paged_ws, c, b, A, 1 << 20, A, 2 * A, 1.0, A, 1 << 20, A, 1 << 30)
    refused(x.kv_read, c, b, A, 2 * A, A, A)
    refused(x.kv_append, c, b, x.KvRows(rows(ld=1 << 20), rows(ld=1 << 20), rows(ld=1 << 20)), A, 2 * A, A)


@pytest.mark.parametrize("bad", BAD_BATCH, ids=str)
def test_bad_batches(bad):
    c, b = cfg(), batch(**bad)
    refused(x.attn_paged_ws, c, b, A, 1024, A, 2 * A, 1.0, A, 1024, A, 1 << 30)
    refused(x.attn_paged, c, b, A, 1024, A, 2 * A, 1.0, A, 1024)
    refused(x.kv_read, c, b, A, 2 * A, A, A)
    refused(x.kv_append, c, b, x.KvRows(rows(), rows(), rows()), A, 2 * A, A)


def test_bad_attention_arguments():
    c, b = cfg(), batch(max_kv=100000, table_ld=2000)
    good = [A, 1024, A, 2 * A, 0.1, A, 1024]
    for i, v in [(0, None), (0, A + 8), (1, 1023), (1, 1020), (1, 1028), (2, None), (2, A + 128), (3, None), (3, A),
                 (4, 0.0), (4, -1.0), (4, float("nan")), (4, float("inf")), (5, None), (5, A + 4), (6, 512)]:
        a = list(good)
        a[i] = v
        refused(x.attn_paged_ws, c, b, *a, A, 1 << 40)
    need = x.attn_paged_workspace_bytes(c, b)
    assert need > 0
    refused(x.attn_paged_ws, c, b, *good, None, need)
    refused(x.attn_paged_ws, c, b, *good, A, need - 1)
    refused(x.attn_paged_ws, c, b, *good, A + 128, need)


def test_bad_append_arguments():
    c, b = cfg(), batch()
    ok = lambda **k: rows(**k)  # noqa: E731
    for r in [x.KvRows(ok(), ok(t=x.T_F16), ok()), x.KvRows(ok(p=None), ok(), ok()), x.KvRows(ok(ld=1020), ok(), ok()),
              x.KvRows(ok(), ok(ld=255), ok()), x.KvRows(ok(), ok(p=A + 4), ok()), x.KvRows(ok(), ok(), ok(ld=4097)),
              x.KvRows(ok(t=7), ok(t=7), ok(t=7)), x.KvRows(ok(rs=A), ok(), ok()),
              x.KvRows(ok(t=x.T_I32), ok(t=x.T_I32), ok(t=x.T_I32)),
              x.KvRows(ok(), ok(), ok(), A, A, -1.0), x.KvRows(ok(), ok(), ok(), None, A, float("nan")),
              x.KvRows(ok(), ok(), ok(), None, None, 0.0, A, 99), x.KvRows(ok(), ok(), ok(), None, None, 0.0, A + 4, 100)]:
        refused(x.kv_append, c, b, r, A, 2 * A, A)
    r = x.KvRows(ok(), ok(), ok())
    refused(x.kv_append, c, b, r, A, 2 * A, None)      # queries without a place for them
    refused(x.kv_append, c, b, r, A, 2 * A, A + 8)
    refused(x.kv_append, c, b, r, A, A, A)
    refused(x.kv_append, c, b, r, None, A, A)
    refused(x.kv_read, c, b, A, 2 * A, None, A)
    refused(x.kv_read, c, b, A, 2 * A, A, A + 2)
    for a in [(96, 10, 1e6, A), (128, -1, 1e6, A), (128, 10, 0.0, A), (128, 10, float("inf"), A), (128, 10, 1e6, None),
              (128, 10, 1e6, A + 8)]:
        refused(x.rope_table, *a)


def test_bad_rows_arguments():
    for n, d, r in [(-1, 64, rows()), (1, 0, rows()), (1, x.ROWS_MAX_D + 1, rows(ld=1 << 20)), (1, 64, rows(ld=63)),
                    (1, 64, rows(p=None)), (1, 64, rows(p=A + 2)), (1, 64, rows(t=2)), (1, 64, rows(rs=A)),
                    (1, 64, rows(t=x.T_I32, rs=A)), (1, 64, rows(t=x.T_I32, cs=A)), (1 << 24, 64, rows())]:
        refused(x.quant_i8, n, d, r, A, A)
        refused(x.add_rmsnorm_i8, n, d, r, None, A, 1e-6, None, 0, A, A)
    refused(x.quant_i8, 1, 64, rows(), None, A)
    refused(x.quant_i8, 1, 64, rows(), A, A + 2)
    refused(x.add_rmsnorm_i8, 1, 64, rows(t=x.T_I32, rs=A, cs=A), None, A, 1e-6, None, 0, A, A)
    refused(x.add_rmsnorm_i8, 1, 64, rows(), None, None, 1e-6, None, 0, A, A)
    refused(x.add_rmsnorm_i8, 1, 64, rows(), None, A, -1e-6, None, 0, A, A)
    refused(x.add_rmsnorm_i8, 1, 64, rows(), rows(), A, 1e-6, None, 64, A, A)
    refused(x.add_rmsnorm_i8, 1, 64, rows(), rows(), A, 1e-6, A, 63, A, A)
    refused(x.add_rmsnorm_i8, 1, 64, rows(), rows(), A, 1e-6, A, 64, A, A)      # in place with another stride
    refused(x.add_rmsnorm_i8, 1, 64, rows(), rows(t=x.T_I32), A, 1e-6, 2 * A, 64, A, A)


def test_nothing_to_do_is_no_error():
    c = cfg()
    for b in (batch(n_seq=0, q_start=None, kv_len=None, block_table=None), batch(n_rows=0, q_start=None, kv_len=None,
                                                                                 block_table=None)):
        assert x.attn_paged_workspace_bytes(c, b) == 0
        x.attn_paged_ws(c, b, A, 1024, A, 2 * A, 0.1, A, 1024, None, 0)
        x.kv_read(c, b, A, 2 * A, A, A)
        x.kv_append(c, b, x.KvRows(rows(), rows(), rows()), A, 2 * A, A)
    x.quant_i8(0, 64, rows(), A, A)
    x.add_rmsnorm_i8(0, 64, rows(), None, A, 1e-6, None, 0, A, A)
    x.rope_table(128, 0, 1e6, A)


def test_pool_sizes():
    assert x.kv_pool_bytes(cfg()) == 4 * 2 * 64 * 80
    assert x.kv_pool_bytes(cfg(kv_type=x.T_BF16)) == 4 * 2 * 64 * 256
    assert x.kv_pool_bytes(cfg(head_dim=64, page=16, act_type=x.T_F16)) == 4 * 2 * 16 * 40
    assert x.kv_pool_bytes(cfg(n_pages=1 << 22, kv_type=x.T_BF16)) == (1 << 22) * 2 * 64 * 256   # past 32 bits


def test_structures_match_the_header():
    """Sizes and offsets that a C compiler gives the header's structures (x86-64)."""
    assert ctypes.sizeof(x.Rows) == 40 and x.Rows.ld.offset == 16
    assert ctypes.sizeof(x.KvCfg) == 28
    assert ctypes.sizeof(x.KvBatch) == 48 and x.KvBatch.q_start.offset == 24
    assert ctypes.sizeof(x.KvRows) == 160 and x.KvRows.eps.offset == 136 and x.KvRows.rope.offset == 144


@pytest.mark.parametrize("kv", [ref.F16, ref.BF16, ref.Q4])
@pytest.mark.parametrize("hd", [64, 128])
def test_layout_round_trip(kv, hd):
    g = np.random.default_rng(3)
    c = ref.Cache(4, 2, hd, 16, 3, ref.BF16 if kv == ref.BF16 else ref.F16, kv)
    K, V = (g.standard_normal((3, 2, 16, hd)).astype(np.float32) for _ in range(2))
    kb, vb = c.encode(K, V)
    assert kb.size == vb.size == x.kv_pool_bytes(x.KvCfg(4, 2, hd, 16, 3, c.act, kv))
    k, v = c.decode(kb, vb)
    if kv == ref.Q4:
        for a, b in ((K, k), (V, v)):
            t = a.reshape(-1, 32)
            # half a step of the codes, 15 steps' rounded step, the minimum's and the value's fp16 rounding
            st = (t.max(1) - t.min(1)) / 15
            bound = st * (0.5 + 16 * 2.0 ** -11) + 3 * 2.0 ** -11 * np.abs(t).max(1)
            assert (np.abs(t - b.reshape(-1, 32)).max(1) <= bound).all()
    else:
        # below 2^-14 fp16 has steps of 2^-24, so a rounding is off by at most 2^-25 there
        u, tiny = ref.HALF_STEP[kv], 2.0 ** -25 if kv == ref.F16 else 0.0
        assert (np.abs(k - K) <= u * np.abs(K) + tiny).all() and (np.abs(v - V) <= u * np.abs(V) + tiny).all()
