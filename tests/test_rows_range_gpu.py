"""x100_add_rmsnorm_i8_hip at the ends of fp32's range, and with eps = 0."""
import numpy as np
import pytest
import torch

import paged_ref as ref
import x100hip as x
from test_rows_gpu import check, stream

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [1, 8, 100, 513, 2048, 4104, 16384])
@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-6, 3.0])
@pytest.mark.parametrize("with_delta", [False, True])
def test_rows_of_any_size(dev, d, eps, with_delta):
    g = np.random.default_rng(d)
    sizes = [0.0, 1e-44, 1e-38, 1e-31, 1e-30, 1e-24, 1e-19, 1e-10, 1.0, 1e10, 1e18, 1e19, 1e30, 3e37]
    n = len(sizes) + 1
    a = (g.standard_normal((n, d)).clip(-3, 3) * np.array(sizes + [1.0])[:, None]).astype(np.float32)
    a[-1] = np.where(np.arange(d) % 2, np.float32(1e-30), np.float32(2e38))   # squares beyond fp32 beside tiny ones
    w = (1 + 0.1 * g.standard_normal(d)).clip(0.5, 1.5).astype(np.float32)
    h = torch.from_numpy(a).cuda()
    dw = torch.from_numpy(w).cuda()
    q, sc = torch.full((n, d), 99, dtype=torch.int8, device=dev), torch.full((n,), 7.0, device=dev)
    rows = x.Rows(ref.F32, h.data_ptr(), d, None, None)
    zero = torch.zeros(n, d, device=dev)
    delta = x.Rows(ref.F32, zero.data_ptr(), d, None, None) if with_delta else None
    x.add_rmsnorm_i8(n, d, rows, delta, dw.data_ptr(), eps, h.data_ptr() if with_delta else None, d, q.data_ptr(),
                     sc.data_ptr(), stream())
    torch.cuda.synchronize()
    t = a * w                                                   # in fp32
    assert np.isfinite(t).all() and torch.equal(h.cpu(), torch.from_numpy(a))
    mean = (a.astype(np.float64) ** 2).mean(1) + float(np.float32(eps))
    want, amax = ref.codes_f32(t)
    r = np.where(amax > 0, 1 / np.sqrt(np.where(mean > 0, mean, 1)), 0.0)
    scale = amax.astype(np.float64) * r / 127
    big = scale > 2.0 ** -126                                   # below, fp32 has fewer bits: half a step of 2^-149
    assert np.array_equal(q.cpu().numpy(), want)
    # the mean to fp32, root (halves that), quotient, product, division, power of two
    err = np.abs(sc.cpu().numpy().astype(np.float64) - scale)
    assert (err <= np.where(big, 6 * 2.0 ** -24 * scale, 6 * 2.0 ** -24 * scale + 2.0 ** -150)).all(), (err, scale)
    assert not sc[0].item() and not q[0].any()
