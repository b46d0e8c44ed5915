"""Refusals at the limits that x100_rows.h / x100_paged.h state (no GPU: an argument error returns before the device
is looked at; what is within them gets as far as the device)."""
import pytest
import torch

import x100hip as x
from test_paged_args import A, batch, cfg, refused, rows


def test_rows_past_one_launch():
    for n, d, fine in [(1 << 22, 4097, False), (1 << 22, 16384, False), ((1 << 24) - 1, 8192, False), (1 << 24, 1, False),
                       (1 << 24, 4096, False)]:
        refused(x.quant_i8, n, d, rows(ld=1 << 20), A, A)
        refused(x.add_rmsnorm_i8, n, d, rows(ld=1 << 20), None, A, 1e-6, None, 0, A, A)
    if torch.cuda.is_available():
        return
    for n, d in [((1 << 22) - 1, 16384), ((1 << 24) - 1, 4096)]:    # accepted: no device here
        with pytest.raises(x.X100Error) as e:
            x.quant_i8(n, d, rows(ld=1 << 20), A, A)
        assert e.value.code == x.X100_ENODEV


def test_scales_that_are_not_aligned():
    for r in (rows(t=x.T_I32, rs=A + 2, cs=A), rows(t=x.T_I32, rs=A, cs=A + 1)):
        refused(x.quant_i8, 1, 64, r, A, A)
        refused(x.add_rmsnorm_i8, 1, 64, rows(), r, A, 1e-6, 2 * A, 64, A, A)
        refused(x.kv_append, cfg(), batch(), x.KvRows(r, r, r), A, 2 * A, A)


def test_a_scale_that_overflows():
    for scale in (1.1e38, 3.4e38):
        refused(x.attn_paged_ws, cfg(), batch(), A, 1024, A, 2 * A, scale, A, 1024, A, 1 << 30)
        refused(x.attn_paged, cfg(), batch(), A, 1024, A, 2 * A, scale, A, 1024)


def test_batches_past_one_launch_ask_for_no_workspace():
    """Refused before the library's workspace is looked for (here it would have been tebibytes)."""
    many = dict(n_seq=65535, n_rows=(1 << 24) - 1, max_kv=1 << 26, table_ld=1 << 22)
    for c, b in [(cfg(n_head=16, n_head_kv=16, page=16), batch(max_q=1, **many)),       # single tokens in many splits
                 (cfg(n_head=16, n_head_kv=16, page=16), batch(max_q=1 << 20, **many)),  # prompts
                 (cfg(n_head=1024, n_head_kv=1024), batch(n_seq=65535, n_rows=(1 << 24) - 1, max_q=1000, max_kv=16))]:
        w = c.n_head * c.head_dim
        assert x.attn_paged_workspace_bytes(c, b) == 0
        refused(x.attn_paged, c, b, A, w, A, 2 * A, 0.1, A, w)
        refused(x.attn_paged_ws, c, b, A, w, A, 2 * A, 0.1, A, w, A, 1 << 60)
