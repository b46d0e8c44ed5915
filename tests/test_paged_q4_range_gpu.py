"""4-bit groups at the ends of fp16's range: what the append stores reads back finite up to 65504, and as NaN past it."""
import numpy as np
import pytest
import torch

import paged_ref as ref
import x100hip as x
from test_paged_gpu import Setup, TT, stream

pytestmark = pytest.mark.gpu


def encode(t):
    """Codes, d and m of fp32 rows [..., hd] as x100_paged.h gives them, over the whole range."""
    g = np.asarray(t, np.float32).reshape(t.shape[:-1] + (-1, 32))
    lo, hi = g.min(-1), g.max(-1)
    bad = ~(np.abs(g) <= 65504).all(-1)
    with np.errstate(all="ignore"):
        m, d = lo.astype(np.float16), ((hi - lo) * np.float32(1 / 15)).astype(np.float16)
        past = np.isinf((m.astype(np.float64) + 15 * d.astype(np.float64)).astype(np.float16)) & ~bad
        d = np.where(past, (d.view(np.uint16) - past).astype(np.uint16).view(np.float16), d)
        inv = np.where(d > 0, np.float32(1) / d.astype(np.float32), np.float32(0))
        n = np.clip(np.rint((g - m.astype(np.float32)[..., None]) * inv[..., None]), 0, 15)
    n = np.where(bad[..., None], 0, n).astype(np.uint32)
    nan = np.float16(np.nan)
    return n.reshape(t.shape), np.where(bad, nan, d), np.where(bad, nan, m), past


ENDS = [(0, 65504), (-65504, 65504), (-60000, 65500), (-65504, 0), (65504, 65504), (-65504, -65504), (65488, 65504), (65472, 65504),
        (-65480, 65503), (60001, 65504), (-1, 65504), (1e-7, 65504), (0, 65504.004), (0, 65505), (0, 65519), (0, 65520),
        (-65505, 0), (-65519, 3), (0, 1e5), (-1e5, 0), (-3e38, 3e38), (0, 6e-8), (-6e-8, 5e-7), (0, 0)]


@pytest.mark.parametrize("act", [ref.F16, ref.BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("rows", [[8 * 40], [3, 5, 9, 1, 303]], ids=str)
def test_groups_at_the_ends(dev, act, hd, rows):
    s = Setup(70, 1, 1, hd, 32, act, ref.Q4, rows, rows)
    g, n = s.g, s.n_rows
    lo, hi = (np.array([e[i] for e in ENDS], np.float32) for i in (0, 1))
    near = g.integers(0, 2, (n, 2, hd // 32)) == 0     # half of the groups: limits and values near 65504
    which = g.integers(0, len(ENDS), near.shape)
    a = np.where(near, np.float32(-1) * g.integers(0, 65505, near.shape), lo[which])[..., None]
    b = np.where(near, 65504 - g.integers(0, 40, near.shape), hi[which])[..., None]
    t = (a + (b - a) * g.random(near.shape + (32,))).astype(np.float32)
    t = np.clip(t, a.astype(np.float32), b.astype(np.float32))
    t[..., 5], t[..., 17] = a[..., 0], b[..., 0]
    t = t.reshape(n, 2, hd)
    d = torch.from_numpy(np.ascontiguousarray(t)).cuda()
    r = x.KvRows(x.Rows(0, None, 0, None, None), *[x.Rows(ref.F32, d.data_ptr() + 4 * hd * i, 2 * hd, None, None) for i in (0, 1)])
    x.kv_append(s.cfg, s.batch, r, s.dk.data_ptr(), s.dv.data_ptr(), None, stream())
    k, v = (torch.empty((n, hd), dtype=TT[act], device=dev) for _ in range(2))
    x.kv_read(s.cfg, s.batch, s.dk.data_ptr(), s.dv.data_ptr(), k.data_ptr(), v.data_ptr(), stream())
    torch.cuda.synchronize()
    pools = s.c.decode(s.dk.cpu().numpy(), s.dv.cpu().numpy())
    codes, dd, mm, past = encode(t)
    want = ref.q4_values(codes, dd, mm)
    fits = (np.abs(t.reshape(n, 2, -1, 32)) <= 65504).all(-1).repeat(32, -1).reshape(t.shape)
    assert past.any() and (~fits).any() and np.isfinite(want[fits]).all() and np.isnan(want[~fits]).all()
    # half a step, the steps' and the value's rounding, and where d is the fp16 below, 15 times its last place
    step = dd.astype(np.float64).repeat(32, -1).reshape(t.shape)
    bound = 0.5 * step + 16 * 2.0 ** -10 * step + 3 * 2.0 ** -11 * np.abs(t) + 2.0 ** -24 * 16
    assert (np.abs(want - t)[fits] <= bound[fits]).all()
    for i in range(len(rows)):
        for j in range(rows[i]):
            row, at = int(s.q_start[i]) + j, (s.table[i][j // 32], 0, j % 32)
            for got, out, w in ((pools[0], k, 0), (pools[1], v, 1)):
                assert np.array_equal(got[at], want[row, w], equal_nan=True), (row, w)
                held = ref.from_bits(ref.to_bits(want[row, w], act), act)
                assert np.array_equal(out[row].float().cpu().numpy(), held.astype(np.float32), equal_nan=True), (row, w)
