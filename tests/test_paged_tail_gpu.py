"""Attention over the paged cache where one position outweighs a long tail of small weights (as an attention sink does):
the tail's share is kept."""
import numpy as np
import pytest

import paged_ref as ref
from test_paged_gpu import Setup, kinds

pytestmark = pytest.mark.gpu


@kinds
@pytest.mark.parametrize("bits", [16.3, 22.0, 25.0, 25.4, 28.7, 30.9])
@pytest.mark.parametrize("q_lens,kv_lens", [([1], [300]), ([1] * 70, [4000] * 70), ([1], [60001]), ([40], [500]), ([33], [16000]),
                                            ([40, 1, 1, 1], [6000, 5000, 100, 4096])], ids=str)
def test_a_long_tail_beside_a_peak(dev, act, kv, bits, q_lens, kv_lens):
    s = Setup(80, 2, 1, 64, 64, act, kv, q_lens, kv_lens)
    c, scale = s.c, 0.125
    K, V = np.zeros((c.n_pages, 1, 64, 64), np.float32), np.zeros((c.n_pages, 1, 64, 64), np.float32)
    V[:] = 1 + 0.5 * s.g.random((1, 1, 1, 64)).astype(np.float32)       # the tail's values: the same at every position
    for i in range(len(kv_lens)):
        first = s.table[i][0]
        K[first, 0, 0, 0] = 8.0                                         # the peak: position 0, with V = 0
        V[first, 0, 0] = 0.0
    s.kb, s.vb = c.encode(K, V)
    s.upload()
    dq, q = s.queries()
    dq.zero_()
    q[:] = 0
    part = ref.to_bits(np.float32([bits * np.log(2.0)]), act)           # 8 * q * scale = q
    dq[:, 0] = dq[:, 64] = int(part.view(np.int16)[0])
    q[:, :, 0] = ref.from_bits(part, act)[0]
    out = s.attend(dq, 128, scale).float().cpu().numpy().astype(np.float64).reshape(s.n_rows, 2, 64)
    K, V = c.decode(s.kb, s.vb)
    w = np.exp(-q[0, 0, 0] * K[s.table[0][0], 0, 0, 0] * scale)         # of a tail position
    tail = V[s.table[0][0], 0, 1]
    u_p, u_out = ref.HALF_STEP[ref.F16 if kv == ref.Q4 else act], ref.HALF_STEP[act]
    for i, L in enumerate(kv_lens):
        for j in range(q_lens[i]):
            n = L - q_lens[i] + j                                       # tail positions of the row
            share = n * w / (1 + n * w)
            want = share * tail
            # a weight is off by half a step, of fp16 at least 2^-25 at a lift of 2^7 (2^4: prompts); its exponent by
            # 2^-20; the peak's by half a step; n sums in fp32; the result's rounding, of fp16 at least 2^-25
            each = max(u_p, 2.0 ** (-32 if max(q_lens) == 1 else -29) / w) if u_p < 2.0 ** -8 else u_p
            tol = (each + u_p + 2.0 ** -20 * 20 + n * 2.0 ** -24 + u_out * 1.01) * want + 2.0 ** -25 * (act == ref.F16)
            d = np.abs(out[int(s.q_start[i]) + j] - want)
            assert (d <= tol).all(), (i, j, d.max(), want.max())
