"""Plain forms of x100_sparse.h for the tests, in 64 bits."""
import numpy as np

import paged_ref as ref


def rows_of(q_start, kv_len, n_rows, max_q, max_kv):
    """(row, sequence, position) of every row of a sequence that keeps the bounds."""
    for s in range(len(kv_len)):
        q0, q1, L = int(q_start[s]), int(q_start[s + 1]), int(kv_len[s])
        if 0 <= q0 <= q1 <= n_rows and q1 - q0 <= max_q and 0 <= L <= max_kv:
            for r in range(q0, q1):
                yield r, s, L - (q1 - q0) + r - q0


def means(cache, K, rows, table, old):
    """old: 16-bit patterns [n_pages][n_kv][hd]; those of the pages that the rows complete are made anew."""
    new = old.copy()
    for r, s, pos in rows:
        if pos >= 0 and pos % cache.page == cache.page - 1:
            pg = int(table[s][pos // cache.page])
            if 0 <= pg < cache.n_pages:
                new[pg] = ref.to_bits((K[pg].sum(1) / cache.page).astype(np.float32), cache.act)
    return new


def select(cache, q, mean, rows, table, n_sel, n_first, n_last, out):
    """out [n_rows][n_kv][n_sel] in place; q [n_rows][n_head][hd], mean [n_pages][n_kv][hd] float64."""
    G = cache.n_head // cache.n_kv
    for r, s, pos in rows:
        out[r] = -1
        if pos < 0:
            continue
        own = pos // cache.page
        pg = np.asarray(table[s][:own + 1])
        ok = (pg >= 0) & (pg < cache.n_pages)
        b = np.arange(own + 1)
        always = (b < n_first) | (b > own - n_last)
        for h in range(cache.n_kv):
            with np.errstate(all="ignore"):
                sc = mean[np.where(ok, pg, 0), h] @ q[r, h * G:(h + 1) * G].sum(0)
            sc = np.where(np.isnan(sc), -np.inf, sc)
            order = sorted(b[ok], key=lambda i: (not always[i], 0 if always[i] else -sc[i], i))
            best = sorted(order[:n_sel])
            out[r, h, :len(best)] = best


def list_of(entries, own):
    """The blocks that a list names: up to its first entry that breaks the order."""
    got, last = [], -1
    for e in entries:
        if not last < e <= own:
            break
        got.append(int(e))
        last = e
    return got


def attend(cache, K, V, q, rows, table, sel, scale, out):
    """As paged_ref.attend, over the lists' blocks: out in place, and the bound."""
    G, page = cache.n_head // cache.n_kv, cache.page
    tol = np.zeros_like(out)
    u_out = ref.HALF_STEP[cache.act]
    u_p = ref.HALF_STEP[ref.F16 if cache.kv == ref.Q4 else cache.act]
    tiny = 2.0 ** -25 if cache.act == ref.F16 else 1e-38
    for r, s, pos in rows:
        out[r] = 0
        for kh in range(cache.n_kv):
            see = [(int(table[s][e]), o) for e in list_of(sel[r, kh], pos // page if pos >= 0 else -1)
                   for o in range(min(page, pos - e * page + 1)) if 0 <= table[s][e] < cache.n_pages]
            if not see:
                continue
            pg, off = np.array(see).T
            k, v = K[pg, kh, off], V[pg, kh, off]
            for h in range(kh * G, kh * G + G):
                x = k @ q[r, h] * scale
                top = x.max()
                if top == -np.inf:
                    continue
                with np.errstate(invalid="ignore"):
                    w = np.exp(x - top)
                    w /= w.sum()
                    out[r, h] = w @ v
                    a = w @ np.abs(v)
                    # as in paged_ref.attend
                    es = ((cache.hd + 4) * 2.0 ** -24 * (np.abs(k) @ np.abs(q[r, h]) * scale).max()
                          + 2.0 ** -21 * (1 + np.abs(x).max()))
                    tol[r, h] = (u_p + 2 * es + 2.0 ** -16) * a + u_out * (np.abs(out[r, h]) + u_p * a) + 2.0 ** -24 * np.abs(v).sum(0) + tiny
    return tol
