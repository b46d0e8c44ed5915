"""Plain numpy forms of x100_paged.h / x100_rows.h in 64 bits, and the cache layouts byte by byte."""
import numpy as np

F32, F16, I32, BF16, Q4 = 0, 1, 26, 30, 256
HALF_STEP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}   # relative error of one rounding


def bf16_bits(x):
    """fp32 -> bf16 bits, nearest even (NaN kept)."""
    x = np.ascontiguousarray(x, np.float32)
    u = x.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7fc0), r).astype(np.uint16)


def to_bits(x, t):
    with np.errstate(over="ignore", invalid="ignore"):
        if t == F16:
            return np.asarray(x, np.float32).astype(np.float16).view(np.uint16)
        return bf16_bits(x)


def from_bits(b, t):
    b = np.ascontiguousarray(b, np.uint16)
    if t == F16:
        return b.view(np.float16).astype(np.float64)
    return (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


# ---- 4-bit groups ---------------------------------------------------------------------------------
def q4_encode(x):
    """x [..., hd] fp32 -> codes [..., hd], d and m fp16 [..., hd/32], in fp32 as the header says."""
    x = np.asarray(x, np.float32)
    g = x.reshape(x.shape[:-1] + (-1, 32))
    with np.errstate(all="ignore"):
        lo, hi = g.min(-1), g.max(-1)
        d = ((hi - lo) * np.float32(1 / 15)).astype(np.float16)
        m = lo.astype(np.float16)
        bad = ~(np.isfinite(g).all(-1) & np.isfinite(d) & np.isfinite(m))
        inv = np.where(d > 0, np.float32(1) / d.astype(np.float32), np.float32(0))
        n = np.clip(np.rint((g - m.astype(np.float32)[..., None]) * inv[..., None]), 0, 15)
    n = np.where(bad[..., None], 0, n).astype(np.uint32)
    d, m = np.where(bad, np.float16(np.nan), d), np.where(bad, np.float16(np.nan), m)
    return n.reshape(x.shape), d.astype(np.float16), m.astype(np.float16)


def q4_values(n, d, m):
    """fp16(m + d n), one rounding (the sum is exact in 64 bits), as float64."""
    g = n.reshape(n.shape[:-1] + (-1, 32)).astype(np.float64)
    with np.errstate(invalid="ignore"):
        v = (m.astype(np.float64)[..., None] + d.astype(np.float64)[..., None] * g).astype(np.float16)
    return v.astype(np.float64).reshape(n.shape)


def shift(e):
    return 16 * (e % 2) + 4 * (e // 2)


def words(n):
    """codes [..., 8] -> 32-bit words [...]."""
    w = np.zeros(n.shape[:-1], np.uint32)
    for e in range(8):
        w |= n[..., e].astype(np.uint32) << np.uint32(shift(e))
    return w


def unwords(w):
    return np.stack([(w >> np.uint32(shift(e))) & np.uint32(15) for e in range(8)], -1)


# ---- pools ----------------------------------------------------------------------------------------
class Cache:
    """A configuration's pools on the host: K and V as the numbers they stand for, and their bytes."""

    def __init__(self, n_head, n_kv, hd, page, n_pages, act, kv):
        self.n_head, self.n_kv, self.hd, self.page, self.n_pages, self.act, self.kv = n_head, n_kv, hd, page, n_pages, act, kv

    def encode(self, K, V):
        """K, V [n_pages][n_kv][page][hd] fp32 -> the two pools' bytes."""
        P, H, p, hd = self.n_pages, self.n_kv, self.page, self.hd
        if self.kv != Q4:
            k = to_bits(K, self.kv)
            v = to_bits(V, self.kv).reshape(P, H, p // 8, 8, hd).transpose(0, 1, 2, 4, 3)
            return k.reshape(-1).view(np.uint8), np.ascontiguousarray(v).reshape(-1).view(np.uint8)
        n, d, m = q4_encode(K)
        kb = np.concatenate([words(n.reshape(P, H, p * hd // 8, 8)).view(np.uint8),
                             np.ascontiguousarray(np.stack([d, m], -1)).reshape(P, H, -1).view(np.uint8)], -1)
        n, d, m = q4_encode(V)
        w = words(n.reshape(P, H, p // 8, 8, hd).transpose(0, 1, 2, 4, 3))
        s = np.stack([t.reshape(P, H, p // 8, 8, hd // 32).transpose(0, 1, 2, 4, 3) for t in (d, m)], -2)
        vb = np.concatenate([np.ascontiguousarray(w).reshape(P, H, -1).view(np.uint8),
                             np.ascontiguousarray(s).reshape(P, H, -1).view(np.uint8)], -1)
        return kb.reshape(-1), vb.reshape(-1)

    def decode(self, kb, vb):
        """The pools' bytes -> K, V [n_pages][n_kv][page][hd] float64."""
        P, H, p, hd = self.n_pages, self.n_kv, self.page, self.hd
        if self.kv != Q4:
            k = from_bits(kb.view(np.uint16), self.kv).reshape(P, H, p, hd)
            v = from_bits(vb.view(np.uint16), self.kv).reshape(P, H, p // 8, hd, 8)
            return k, np.ascontiguousarray(v.transpose(0, 1, 2, 4, 3)).reshape(P, H, p, hd)
        c = p * hd // 2
        kb, vb = kb.reshape(P, H, -1), vb.reshape(P, H, -1)
        n = unwords(np.ascontiguousarray(kb[..., :c]).view(np.uint32)).reshape(P, H, p, hd)
        s = np.ascontiguousarray(kb[..., c:]).view(np.float16).reshape(P, H, p, hd // 32, 2)
        k = q4_values(n, s[..., 0], s[..., 1])
        n = unwords(np.ascontiguousarray(vb[..., :c]).view(np.uint32)).reshape(P, H, p // 8, hd, 8)
        n = np.ascontiguousarray(n.transpose(0, 1, 2, 4, 3)).reshape(P, H, p, hd)
        s = np.ascontiguousarray(vb[..., c:]).view(np.float16).reshape(P, H, p // 8, hd // 32, 2, 8)
        d, m = (np.ascontiguousarray(s[..., i, :].transpose(0, 1, 2, 4, 3)).reshape(P, H, p, hd // 32) for i in (0, 1))
        return k, q4_values(n, d, m)


# ---- attention ------------------------------------------------------------------------------------
def attend(cache, K, V, q, q_start, kv_len, table, scale, out, max_q, max_kv):
    """out [n_rows][n_head][hd] float64 in place (refused sequences and rows behind the last left
    alone), and the error bound of a kernel that rounds the weights and the result to 16 bits."""
    n_rows, G = q.shape[0], cache.n_head // cache.n_kv
    tol = np.zeros_like(out)
    u_out = HALF_STEP[cache.act]
    u_p = HALF_STEP[F16 if cache.kv == Q4 else cache.act]
    tiny = 2.0 ** -25 if cache.act == F16 else 1e-38   # half a step of fp16's subnormals
    for s in range(len(kv_len)):
        q0, q1, L = int(q_start[s]), int(q_start[s + 1]), int(kv_len[s])
        if not (0 <= q0 <= q1 <= n_rows and q1 - q0 <= max_q and 0 <= L <= max_kv):
            continue
        pg = np.array([table[s][p // cache.page] for p in range(L)], np.int64)
        ok = (pg >= 0) & (pg < cache.n_pages)
        off = np.arange(L) % cache.page
        for r in range(q0, q1):
            pos = L - (q1 - q0) + r - q0
            see = np.nonzero(ok[:pos + 1])[0] if pos >= 0 else np.zeros(0, np.int64)
            for h in range(cache.n_head):
                kh = h // G
                if not len(see):
                    out[r, h] = 0
                    continue
                k, v = K[pg[see], kh, off[see]], V[pg[see], kh, off[see]]
                x = k @ q[r, h] * scale
                top = x.max()
                if top == -np.inf:
                    out[r, h] = 0
                    continue
                with np.errstate(invalid="ignore"):
                    w = np.exp(x - top)
                    w /= w.sum()
                    out[r, h] = w @ v
                    a = w @ np.abs(v)
                    # a score is a sum of hd fp32 products; its error is the weight's relative error (of
                    # the row's weight and of the others'), as are the rescaled exponent's roundings
                    es = ((cache.hd + 4) * 2.0 ** -24 * (np.abs(k) @ np.abs(q[r, h]) * scale).max()
                          + 2.0 ** -21 * (1 + np.abs(x).max()))
                    tol[r, h] = (u_p + 2 * es + 2.0 ** -16) * a + u_out * (np.abs(out[r, h]) + u_p * a) + 2.0 ** -24 * np.abs(v).sum(0) + tiny
    return tol


# ---- append ---------------------------------------------------------------------------------------
def rotate(x, pos, base):
    """x [..., hd] at position pos (float64)."""
    hd = x.shape[-1]
    a = pos * float(base) ** (-np.arange(0, hd, 2) / hd)
    c, s = np.cos(a), np.sin(a)
    lo, hi = x[..., :hd // 2], x[..., hd // 2:]
    return np.concatenate([lo * c - hi * s, lo * s + hi * c], -1)


def head_norm(x, w, eps):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w


# ---- int8 rows ------------------------------------------------------------------------------------
def codes_f32(t):
    """Codes and amax of rows t (fp32 values), in fp32 as the header says: bit for bit."""
    t = np.asarray(t, np.float32)
    with np.errstate(all="ignore"):
        amax = np.abs(t).max(1)
        fin = np.isfinite(t).all(1)
        some = fin & (amax >= np.float32(2.0 ** -100))
        inv = np.where(some, np.float32(127) * (np.float32(1) / amax), np.float32(0)).astype(np.float32)
        c = np.rint(t * inv[:, None])
    c = np.where(some[:, None], c, 0).astype(np.int8)
    return c, np.where(some, amax, np.where(fin, np.float32(0), np.float32(np.nan)))
