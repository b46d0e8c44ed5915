"""Plain forms of x100_fp8.h for the tests: rows to e4m3 codes and scales, and the product in 64 bits."""
import numpy as np
import torch

E4M3 = torch.float8_e4m3fn
TT = {0: torch.float32, 1: torch.float16, 30: torch.bfloat16}
STEP = {0: 2.0 ** -24, 1: 2.0 ** -11, 30: 2.0 ** -8}    # half a step of a type, relative
LOW = {0: 2.0 ** -149, 1: 2.0 ** -25, 30: 2.0 ** -134}  # half a step at the bottom of its range (fp32: a whole one)


def blocks(n):
    return -(-n // 128)


def codes(t):
    """t [n, d] fp32 -> (codes uint8 [n, d up to 16], amax fp32 [n, blocks], finite [n, blocks])."""
    n, d = t.shape
    nb, dp = blocks(d), -(-d // 16) * 16
    g = np.zeros((n, nb * 128), np.float32)
    g[:, :d] = t
    g = g.reshape(n, nb, 128)
    ok = np.isfinite(g).all(2)
    amax = np.where(ok, np.abs(np.where(np.isfinite(g), g, 0)).max(2), 0).astype(np.float32)
    some = ok & (amax >= 2.0 ** -100)
    with np.errstate(divide="ignore", over="ignore"):
        f = np.where(some, np.float32(448) * (np.float32(1) / amax), np.float32(0)).astype(np.float32)
    y = np.where(some[..., None], np.where(np.isfinite(g), g, 0) * f[..., None], 0).astype(np.float32)
    c = torch.from_numpy(y).to(E4M3).view(torch.uint8).numpy()
    c = np.where(some[..., None], c, 0).reshape(n, -1)[:, :dp].astype(np.uint8)
    return c, np.where(some, amax, np.float32(0)), ok


def values(c):
    """uint8 codes (numpy) -> float64."""
    return torch.from_numpy(np.ascontiguousarray(c)).view(E4M3).double().numpy()


def product(a, sa, w, sw):
    """Codes a [M, K], w [N, K], scales sa [blocks, M], sw [blocks of N, blocks]: (C, sum of the terms' sizes), fp64."""
    M, K = a.shape
    N = w.shape[0]
    A, W = torch.from_numpy(values(a)), torch.from_numpy(values(w))
    c, size = torch.zeros(M, N, dtype=torch.float64), torch.zeros(M, N, dtype=torch.float64)
    col = np.arange(N) // 128
    for b in range(blocks(K)):
        k = slice(128 * b, min(128 * b + 128, K))
        s = torch.from_numpy(sa[b].astype(np.float64))[:, None] * torch.from_numpy(sw[:, b].astype(np.float64)[col])
        c += (A[:, k] @ W[:, k].T) * s
        size += (A[:, k].abs() @ W[:, k].abs().T) * s.abs()
    return c.numpy(), size.numpy()


def product_bound(K, c, size, c_type, cut=None):
    """How far a product may be off.  In fp32: 128 additions in a block that may each cut instead of round (two half steps),
    one addition per block and the two scales' products, then the store's rounding.
    cut (16-bit results): the sum over groups of 8 neighbouring k of the largest term's size, or any larger number.  The
    matrix cores add the products of such a group in fixed point and cut what lies below 2^-13 of the power of two
    under the largest, so each of the 7 others loses less than 2^-13 of the largest."""
    f32 = (2 * 128 + blocks(K) + 4) * 2.0 ** -24 * size
    if c_type != 0:
        f32 = f32 + 7 * 2.0 ** -13 * (size if cut is None else cut)
    return f32 + (np.abs(c) + f32) * STEP[c_type] + LOW[c_type]


def group_largest(a, sa, w, sw, m, n):
    """Of the outputs (m[i], n[i]): the sum over groups of 8 neighbouring k of the largest term's size."""
    A, W = np.abs(values(a[m])), np.abs(values(w[n]))
    K = A.shape[1]
    top = (A * W).reshape(len(m), K // 8, 8).max(2)
    s = np.abs(sa.astype(np.float64)[:, m].T * sw.astype(np.float64)[n // 128])
    return (top * np.repeat(s, 16, 1)[:, :K // 8]).sum(1)
