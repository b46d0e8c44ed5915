"""Attention over the paged cache where scores are NaN: a row that attends to one gives NaN, however the positions are
spread over waves, splits and kernels, and no other row does."""
import numpy as np
import pytest

import paged_ref as ref
from test_paged_gpu import Setup, compare, kinds

pytestmark = pytest.mark.gpu

# rows and positions of the sequences: single tokens in one split and in many (more than a block per head joins), and
# prompts in one and in several
SHAPES = [([1, 1, 1, 1], [1, 5, 40, 300]), ([1, 2], [900, 3000]), ([1], [9000]), ([40, 33], [40, 90]), ([70], [3000]),
          ([70, 1, 1], [2600, 2000, 7])]


@kinds
@pytest.mark.parametrize("q_lens,kv_lens", SHAPES, ids=[str(s) for s in SHAPES])
@pytest.mark.parametrize("where", ["query", "every key", "first 32", "first 128", "last", "one"])
def test_scores_that_are_nan(dev, act, kv, q_lens, kv_lens, where):
    s = Setup(60, 4, 2, 64, 16, act, kv, q_lens, kv_lens)
    c = s.c
    K, V = c.decode(s.kb, s.vb)
    for i, L in enumerate(kv_lens):
        at = {"every key": range(L), "first 32": range(min(32, L)), "first 128": range(min(128, L)), "last": [L - 1],
              "one": [L // 2], "query": []}[where]
        for p in at:   # of one KV head, one element
            K[s.table[i][p // 16], 1, p % 16, 3 + p % 50] = np.nan
    s.kb, s.vb = c.encode(K.astype(np.float32), V.astype(np.float32))
    s.upload()
    dq, q = s.queries()
    if where == "query":
        rows = [int(r) for r in s.q_start[:-1]] + [s.n_rows - 1]
        dq[rows, 2 * 64 + 5] = 0x7fff            # a NaN of either type, in one head
        q[rows, 2, 5] = np.nan
    out = s.attend(dq, 256, 0.125).float().cpu().numpy().astype(np.float64).reshape(s.n_rows, 4, 64)
    want, tol = s.expected(q, 0.125)
    assert np.isnan(want).any() and np.isfinite(want).any()
    compare(out, want, tol)
