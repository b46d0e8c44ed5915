"""Operators of a served batch: matrix product in 8-bit floating point (e4m3) with a scale per block of 128, the rows it
takes (plain rows, residual + RMSNorm), and sparse attention over the paged KV cache (block means and the selection
of blocks per query, attention over the selected blocks).

Each case is one call (or the calls a program makes together) on device tensors.  Lengths of ragged
batches follow from the case alone; values, page numbers and weights from the seed.  Layouts and formulas are those of
include/x100_fp8.h, include/x100_sparse.h and include/x100_paged.h.

  python3 -c "import sys; sys.path.insert(0, 'perf'); import more_operators as o; print(o.listed())"
"""
import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
E4M3 = torch.float8_e4m3fn
# bit position of element e of 8 in a 32-bit word of 4-bit codes: even elements in the low half
SHIFT = [0, 16, 4, 20, 8, 24, 12, 28]
EPS = 1e-6
N_FIRST, N_LAST = 1, 2     # blocks that every query takes: the first one, its own and the one before


def _case(name, **kw):
    return dict({"name": name}, **kw)


HEADS = dict(n_head=32, n_kv=4, hd=128)     # 32 query heads on 4 KV heads of 128


def listed():
    return [
        # one user: the q, k and v projections of a new token
        _case("linear 1x5120x2048", op="gemm", M=1, N=5120, K=2048, out="bf16"),
        # a server's decode step: the output projection of 64 tokens
        _case("linear 64x2048x4096", op="gemm", M=64, N=2048, K=4096, out="bf16"),
        # logits of a few tokens
        _case("lm_head 8x151936x2048", op="gemm", M=8, N=151936, K=2048, out="f32"),
        # prompts of several users in one batch: q, k and v
        _case("linear 16381x5120x2048", op="gemm", M=16381, N=5120, K=2048, out="bf16"),
        # residual and norm in front of the projections: a decode step, and a prompt
        _case("norm 64x2048 bf16", op="norm", rows=64, d=2048, x="bf16", delta="bf16"),
        _case("norm 16381x2048 f32 bf16", op="norm", rows=16381, d=2048, x="f32", delta="bf16"),
        # the attention's output in front of the output projection
        _case("quant 16x4096 bf16", op="quant", rows=16, d=4096, x="bf16"),
        _case("quant 16384x4096 f16", op="quant", rows=16384, d=4096, x="f16"),
        # which blocks the new tokens of 16 long contexts attend to; the rows of a prompt's piece behind a long prefix
        _case("select 16x1 on 60032", op="select", n_seq=16, q=1, kv=60032, page=64, act="bf16", cache="bf16",
              n_sel=32, **HEADS),
        _case("select 1x2001 on 32000 q4", op="select", n_seq=1, q=2001, kv=32000, page=64, act="f16", cache="q4",
              n_sel=32, **HEADS),
        # the attention over them
        _case("sparse 16x1 on 60032", op="sparse", n_seq=16, q=1, kv=60032, page=64, act="bf16", cache="bf16",
              n_sel=32, **HEADS),
        _case("sparse 2x1013 on 16384 q4", op="sparse", n_seq=2, q=1013, kv=16384, page=64, act="f16", cache="q4",
              n_sel=16, **HEADS),
    ]


def _logint(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["gemm", "gemm", "gemm", "norm", "quant", "select", "sparse", "sparse"])
    if op == "gemm":
        K = 16 * _logint(rng, 8, 1024)
        N = rng.choice([_logint(rng, 16, 16000), 128 * _logint(rng, 1, 125), 16 * _logint(rng, 4, 8000)])
        N = min(N, 300000000 // K)
        M = _logint(rng, 1, max(1, min(16000, int(1.7e11 / (N * K)), 80000000 // N)))
        return dict(op=op, M=M, N=N, K=K, out=rng.choice(["f32", "f16", "bf16", "bf16"]))
    if op in ("norm", "quant"):
        d = rng.choice([_logint(rng, 64, 8192), 16 * _logint(rng, 16, 512), 512, 1024, 2048, 4096])
        c = dict(op=op, rows=_logint(rng, 1, max(1, min(16000, 32000000 // d))), d=d, x=rng.choice(["f32", "f16", "bf16"]))
        if op == "norm":
            c["delta"] = rng.choice(["f32", "f16", "bf16", "bf16", "none"])
        return c
    hd = rng.choice([64, 128, 128])
    n_kv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 8, 8, 16]) if n_kv <= 4 else rng.choice([1, 2, 4])
    act, page = rng.choice(["f16", "bf16"]), rng.choice([16, 32, 64, 64, 128])
    n_sel = _logint(rng, 4, 64)
    c = dict(op=op, n_head=n_kv * group, n_kv=n_kv, hd=hd, page=page, act=act, cache=rng.choice([act, "q4"]), n_sel=n_sel)
    kv = _logint(rng, 16, 60000)
    q = rng.choice([1, 1, _logint(rng, 1, min(kv, 2000))])
    # rows times what each gathers, scores of all blocks, and the cache itself
    most = min(256, 530000000 // (q * n_kv * n_sel * page * hd), 130000000 // (q * n_kv * (kv // page + 1)),
               900000 * 512 // (kv * n_kv * hd))
    while most < 1:
        q = (q + 1) // 2
        most = 1 if q == 1 else 530000000 // (q * n_kv * n_sel * page * hd)
    return dict(c, n_seq=_logint(rng, 1, most), q=q, kv=max(4, kv))


def _lengths(case):
    """(q_len, kv_len) of every sequence: the first has the case's full lengths, the others less."""
    r = random.Random("%d %d %d" % (case["n_seq"], case["q"], case["kv"]))
    q, kv = case["q"], case["kv"]
    ql, kl = [q], [kv]
    for i in range(1, case["n_seq"]):
        a = q if q <= 4 else (1 if i % 4 == 3 else r.randint(max(1, q // 4), q))
        cached = kv - q
        ql.append(a)
        kl.append(a + (r.randint(cached // 4, cached) if cached else 0))
    return ql, kl


def _blocks(n):
    return -(-n // 128)


def _completed(case):
    """Pages that each sequence's new rows complete: [first, last)."""
    page = case["page"]
    return [((k - a) // page, k // page) for a, k in zip(*_lengths(case))]


def work(case):
    if case["op"] == "gemm":
        M, N, K = case["M"], case["N"], case["K"]
        b = M * K + N * K + 4 * (M + _blocks(N)) * _blocks(K) + M * N * SIZE[case["out"]]
        return {"bytes": b, "flops": 2 * M * N * K}
    if case["op"] in ("norm", "quant"):
        n, s = case["rows"] * case["d"], SIZE[case["x"]]
        b = n * (s + 1) + 4 * case["rows"] * _blocks(case["d"])
        if case["op"] == "quant":
            return {"bytes": b, "flops": 3 * n}
        t = case["delta"]
        return {"bytes": b + 4 * case["d"] + (0 if t == "none" else n * (SIZE[t] + s)), "flops": 6 * n}
    ql, kl = _lengths(case)
    page, hd, kv, nh, n_sel = case["page"], case["hd"], case["n_kv"], case["n_head"], case["n_sel"]
    per = hd * (2.0 if case["cache"] != "q4" else 0.625)     # bytes of a K (or V) head row
    rows = sum(ql)
    if case["op"] == "select":
        done = sum(b - a for a, b in _completed(case))
        blocks = sum((k - 1) // page for k in kl)
        scored = sum(sum(p // page for p in range(k - a, k)) for a, k in zip(ql, kl))
        return {"bytes": kv * (done * (page * per + 2 * hd) + blocks * 2 * hd + rows * n_sel * 4) + 2 * rows * nh * hd,
                "flops": 2 * scored * kv * hd}
    pages, seen = 0, 0
    for a, k in zip(ql, kl):
        pages += min((k - 1) // page + 1, a * n_sel)
        for p in range(k - a, k):
            seen += min(n_sel - 1, p // page) * page + p % page + 1
    return {"bytes": pages * page * kv * 2 * per + 2 * rows * nh * hd * 2 + rows * kv * n_sel * 4,
            "flops": 4 * seen * nh * hd}


# ---- the cache's pages ----------------------------------------------------------------------------

def _pages(case, pool, which, at, head):
    """Values of pages `at` at KV heads `head` (index tensors of one shape): [..., page, hd] fp32."""
    kv, page, hd = case["n_kv"], case["page"], case["hd"]
    if case["cache"] != "q4":
        t = pool.view(TORCH[case["cache"]])
        if which == "k":
            return t.view(-1, kv, page, hd)[at, head].float()
        t = t.view(-1, kv, page // 8, hd, 8)[at, head].float()
        return t.transpose(-1, -2).reshape(*at.shape, page, hd)
    b = pool.view(-1, kv, page * hd * 5 // 8)[at, head]
    c, s = b[..., :page * hd // 2].contiguous().view(torch.int32), b[..., page * hd // 2:].contiguous().view(torch.float16)
    sh = torch.tensor(SHIFT, device=pool.device, dtype=torch.int32)
    c = ((c[..., None] >> sh) & 15).to(torch.uint8)          # [..., words, 8]
    if which == "k":
        c = c.reshape(*at.shape, page, hd)
        d, m = s.reshape(*at.shape, page, hd // 32, 2).unbind(-1)
    else:
        c = c.reshape(*at.shape, page // 8, hd, 8).transpose(-1, -2).reshape(*at.shape, page, hd)
        s = s.reshape(*at.shape, page // 8, hd // 32, 2, 8)
        d, m = (s[..., i, :].transpose(-1, -2).reshape(*at.shape, page, hd // 32) for i in (0, 1))
    # d n + m in fp32: d n is exact (11 + 4 bits); the sum rounds once more before fp16 only where m
    # and d n are far apart
    g = c.reshape(*at.shape, page, hd // 32, 32).float()
    return (g * d.float()[..., None] + m.float()[..., None]).half().float().reshape(*at.shape, page, hd)


# ---- what a program has in hand -------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed * 1000003 + 29)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    def rand(*shape):
        return torch.rand(*shape, generator=g, device=DEV)

    s = {"case": case}
    if case["op"] == "gemm":
        M, N, K = case["M"], case["N"], case["K"]
        kb = _blocks(K)
        # codes as quantised rows have them: the largest of 128 normal values stands at 448
        for name, n in (("a", M), ("w", N)):
            t = torch.empty(n, K, device=DEV, dtype=torch.bfloat16).normal_(0, 150, generator=g)
            s[name] = t.clamp_(-448, 448).to(E4M3)
            del t
        s["as"] = (0.5 + rand(kb, M)) / 150
        s["ws"] = (0.5 + rand(_blocks(N), kb)) / (150 * math.sqrt(K))
        s["c"] = torch.empty(M, N, dtype=TORCH[case["out"]], device=DEV)
    elif case["op"] in ("norm", "quant"):
        n, d = case["rows"], case["d"]
        s["x"] = (normal(n, d) * (0.5 + 4 * rand(n, 1))).to(TORCH[case["x"]])
        s["q"] = torch.zeros(n, 16 * -(-d // 16), dtype=torch.uint8, device=DEV)
        s["scale"] = torch.empty(_blocks(d), n, device=DEV)
        if case["op"] == "norm":
            s["w"] = 1 + 0.2 * normal(d)
            if case["delta"] != "none":
                s["delta"] = normal(n, d).to(TORCH[case["delta"]])
                s["h"] = torch.empty_like(s["x"])
    else:
        ql, kl = _lengths(case)
        S, page, hd, kv, nh = case["n_seq"], case["page"], case["hd"], case["n_kv"], case["n_head"]
        per = -(-case["kv"] // page)
        n_pages = S * per
        s["table"] = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32).view(S, per).contiguous()
        starts = [0]
        for a in ql:
            starts.append(starts[-1] + a)
        s["q_start"] = torch.tensor(starts, dtype=torch.int32, device=DEV)
        s["kv_len"] = torch.tensor(kl, dtype=torch.int32, device=DEV)
        n = starts[-1]
        s["n_rows"], s["n_pages"] = n, n_pages
        for w in ("k", "v") if case["op"] == "sparse" else ("k",):
            vals = n_pages * kv * page * hd
            if case["cache"] != "q4":
                pool = torch.empty(vals, dtype=TORCH[case["cache"]], device=DEV).normal_(generator=g)
            else:     # random codes with the scales that normal values get: 15 steps over about 4 deviations
                pool = torch.empty(n_pages * kv, page * hd * 5 // 8, dtype=torch.uint8, device=DEV)
                pool[:, :page * hd // 2] = torch.randint(0, 256, (n_pages * kv, page * hd // 2), generator=g,
                                                         device=DEV, dtype=torch.uint8)
                d = 0.25 + 0.1 * rand(n_pages * kv * page * hd // 32)
                m = -7.5 * d + 0.3 * normal(d.numel())
                sc = torch.stack([d, m], -1) if w == "k" else torch.stack([d.view(-1, 8), m.view(-1, 8)], 1)
                pool[:, page * hd // 2:] = sc.half().reshape(n_pages * kv, -1).view(torch.uint8)
            s[w + "_pool"] = pool.view(torch.uint8).reshape(-1)
        # scores of about 1.5 deviations, as heads with normalised queries and keys have them
        s["q"] = (1.5 * normal(n, nh * hd)).to(TORCH[case["act"]])
        if case["op"] == "select":
            s["means"] = (normal(n_pages, kv, hd) / math.sqrt(page)).to(TORCH[case["act"]])
            s["sel"] = torch.empty(n, kv, case["n_sel"], dtype=torch.int32, device=DEV)
        else:
            # lists as the selection gives them; rows near each other mostly want the same blocks
            _, seq, pos = _positions(s)
            own_block = (pos // page)[:, None, None]
            want = (normal(S, kv, per)[seq] + 0.7 * normal(n, kv, per)).double()
            s["sel"] = _choose(want, own_block, case["n_sel"])
            s["out"] = torch.empty_like(s["q"])
    if own:
        _plan(s)
    return s


# ---- the framework's calls ------------------------------------------------------------------------

def _lib():
    here = os.path.join(os.getcwd(), "x100-gemm_amd")
    if here not in sys.path:
        sys.path.insert(0, here)
    import x100hip
    return x100hip


def _plan(s):
    """The descriptors and workspace that a program keeps beside its buffers."""
    x, case = _lib(), s["case"]
    s["lib"] = x
    T = {"f32": x.T_F32, "f16": x.T_F16, "bf16": x.T_BF16, "q4": x.KV_Q4}
    if case["op"] == "gemm":
        s["fa"] = x.Fp8(s["a"].data_ptr(), case["K"], s["as"].data_ptr(), case["M"])
        s["fw"] = x.Fp8(s["w"].data_ptr(), case["K"], s["ws"].data_ptr(), s["ws"].shape[1])
        s["type"] = T[case["out"]]
        return
    if case["op"] in ("norm", "quant"):
        s["rx"] = x.Rows(T[case["x"]], s["x"].data_ptr(), case["d"], None, None)
        s["rd"] = x.Rows(T[case["delta"]], s["delta"].data_ptr(), case["d"], None, None) if "delta" in s else None
        s["fq"] = x.Fp8(s["q"].data_ptr(), s["q"].shape[1], s["scale"].data_ptr(), case["rows"])
        return
    s["cfg"] = x.KvCfg(case["n_head"], case["n_kv"], case["hd"], case["page"], s["n_pages"], T[case["act"]],
                       T[case["cache"]])
    s["batch"] = x.KvBatch(case["n_seq"], s["n_rows"], case["q"], case["kv"], s["table"].shape[1],
                           s["q_start"].data_ptr(), s["kv_len"].data_ptr(), s["table"].data_ptr())
    if case["op"] == "select":
        s["pick"] = x.KvSel(case["n_sel"], N_FIRST, N_LAST)
    else:
        n = x.attn_sparse_workspace_bytes(s["cfg"], s["batch"], case["n_sel"])
        s["ws"] = torch.empty(max(n, 256), dtype=torch.uint8, device=DEV)


def _run_own(s):
    x, case = s["lib"], s["case"]
    stream = torch.cuda.current_stream().cuda_stream
    if case["op"] == "gemm":
        x.gemm_fp8(case["M"], case["N"], case["K"], s["fa"], s["fw"], s["type"], s["c"].data_ptr(), case["N"], stream)
        return s["c"]
    if case["op"] == "quant":
        x.quant_fp8(case["rows"], case["d"], s["rx"], s["fq"], stream)
        return {"codes": s["q"].view(E4M3), "scale": s["scale"]}
    if case["op"] == "norm":
        h = s.get("h")
        x.add_rmsnorm_fp8(case["rows"], case["d"], s["rx"], s["rd"], s["w"].data_ptr(), EPS,
                          None if h is None else h.data_ptr(), case["d"], s["fq"], stream)
        return {"codes": s["q"].view(E4M3), "scale": s["scale"], "h": h}
    w, q = case["n_head"] * case["hd"], s["q"].data_ptr()
    if case["op"] == "select":
        x.kv_means(s["cfg"], s["batch"], s["k_pool"].data_ptr(), s["means"].data_ptr(), stream)
        x.attn_select(s["cfg"], s["batch"], s["pick"], q, w, s["means"].data_ptr(), s["sel"].data_ptr(), stream)
        return {"means": s["means"], "sel": s["sel"]}
    x.attn_sparse_ws(s["cfg"], s["batch"], q, w, s["k_pool"].data_ptr(), s["v_pool"].data_ptr(), case["hd"] ** -0.5,
                     s["sel"].data_ptr(), case["n_sel"], s["out"].data_ptr(), w, s["ws"].data_ptr(), s["ws"].numel(),
                     stream)
    return s["out"]


# ---- the plain forms ------------------------------------------------------------------------------

def _positions(s):
    """Number, sequence and position of every row."""
    r = torch.arange(s["n_rows"], device=DEV)
    seq = torch.searchsorted(s["q_start"][1:].long(), r, right=True)
    return r, seq, s["kv_len"].long()[seq] - s["q_start"].long()[seq + 1] + r


def _choose(score, own_block, n_sel):
    """The n_sel best blocks of score [rows, kv, blocks] (64 bits), ascending, -1 behind them: the first N_FIRST, the
    last N_LAST up to the row's own, then by score, ties to the lowest index."""
    b = torch.arange(score.shape[-1], device=score.device)
    score = torch.where(torch.isnan(score), torch.full_like(score, float("-inf")), score)
    live = (b <= own_block).expand(score.shape)
    forced = ((b < N_FIRST) | (b > own_block - N_LAST)) & live
    # by score, then forced blocks in front and those behind the row's own at the end, each sort keeping the order
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices
    place = torch.where(forced, 0, torch.where(live, 1, 2)).gather(-1, order)
    order = order.gather(-1, torch.sort(place, dim=-1, stable=True).indices)
    best = order[..., :n_sel]
    best = torch.where(live.gather(-1, best), best, score.shape[-1])
    best = torch.sort(best, dim=-1).values
    best = torch.where(best == score.shape[-1], -1, best)
    if best.shape[-1] < n_sel:
        pad = torch.full((*best.shape[:-1], n_sel - best.shape[-1]), -1, device=best.device, dtype=best.dtype)
        best = torch.cat([best, pad], -1)
    return best.to(torch.int32).contiguous()


def _amax(t):
    """Rows t (fp32) -> t in blocks of 128 (zeros behind the end) and their largest sizes [rows, blocks]."""
    n, d = t.shape
    g = torch.nn.functional.pad(t, (0, 128 * _blocks(d) - d)).view(n, -1, 128)
    return g, g.abs().amax(-1)


def _codes(g, amax, width):
    f = 448.0 * (1.0 / amax)
    return (g * f[..., None]).to(E4M3).reshape(g.shape[0], -1)[:, :width].contiguous()


def _run_plain(s):
    case = s["case"]
    if case["op"] == "gemm":
        M, N, K = case["M"], case["N"], case["K"]
        a = s["a"].float() * s["as"].t().repeat_interleave(128, 1)[:, :K]
        w = s["w"].float() * s["ws"].repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]
        return torch.matmul(a, w.t()).to(TORCH[case["out"]])
    if case["op"] == "quant":
        g, amax = _amax(s["x"].float())
        return {"codes": _codes(g, amax, s["q"].shape[1]), "scale": (amax / 448.0).t().contiguous()}
    if case["op"] == "norm":
        x, h = s["x"].float(), None
        if "delta" in s:
            h = (x + s["delta"].float()).to(TORCH[case["x"]])
            x = h.float()
        r = 1.0 / torch.sqrt(x.square().mean(1) + EPS)
        g, amax = _amax(x * s["w"])
        return {"codes": _codes(g, amax, s["q"].shape[1]), "scale": (amax * r[:, None] / 448.0).t().contiguous(), "h": h}
    page, hd, kv, nh, n = case["page"], case["hd"], case["n_kv"], case["n_head"], s["n_rows"]
    act = TORCH[case["act"]]
    r, seq, pos = _positions(s)
    heads = torch.arange(kv, device=DEV)
    if case["op"] == "select":
        # the pages that the rows complete: their last position is a new row
        last = (pos % page == page - 1).nonzero()[:, 0]
        at = s["table"].long()[seq[last], pos[last] // page]
        k = _pages(case, s["k_pool"], "k", at[:, None].expand(-1, kv), heads.expand(len(at), kv))
        s["means"][at] = (k.double().sum(-2) / page).to(act)
        S, q = case["n_seq"], case["q"]
        m = s["means"][s["table"].long()].double().permute(0, 2, 3, 1).contiguous()      # [S, kv, hd, blocks]
        Q = torch.zeros(S, q, kv, hd, device=DEV, dtype=torch.float64)
        i = r - s["q_start"].long()[seq]
        Q[seq, i] = s["q"].double().view(n, kv, nh // kv, hd).sum(2)
        score = torch.matmul(Q.transpose(1, 2).contiguous(), m).transpose(1, 2)[seq, i]   # [rows, kv, blocks]
        return {"means": s["means"], "sel": _choose(score, (pos // page)[:, None, None], case["n_sel"])}
    sel = s["sel"].long()
    block = sel.clamp(min=0)
    at = s["table"].long()[seq[:, None, None], block]                                     # [rows, kv, n_sel]
    place = block[..., None] * page + torch.arange(page, device=DEV)
    hidden = ((sel < 0)[..., None] | (place > pos[:, None, None, None])).view(n, kv, 1, -1)
    who = heads[None, :, None].expand_as(at)
    K = _pages(case, s["k_pool"], "k", at, who).reshape(n, kv, -1, hd)
    sc = torch.matmul(s["q"].float().view(n, kv, nh // kv, hd), K.transpose(-1, -2).contiguous()) * hd ** -0.5
    del K
    sc = sc.masked_fill(hidden, float("-inf"))
    p = (sc - sc.amax(-1, keepdim=True)).exp()
    V = _pages(case, s["v_pool"], "v", at, who).reshape(n, kv, -1, hd)
    return (torch.matmul(p, V) / p.sum(-1, keepdim=True)).reshape(n, nh * hd).to(act)


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the definitions in 64 bits -------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    f8 = torch.float64
    if case["op"] == "gemm":
        c = torch.zeros(case["M"], case["N"], dtype=f8, device=DEV)
        for b in range(_blocks(case["K"])):
            k = slice(128 * b, min(128 * b + 128, case["K"]))
            part = torch.mm(s["a"][:, k].to(f8), s["w"][:, k].to(f8).t().contiguous())
            col = torch.arange(case["N"], device=DEV) // 128
            part *= s["as"][b].to(f8)[:, None]
            part *= s["ws"][:, b].to(f8)[col]
            c += part
        return c
    if case["op"] in ("norm", "quant"):
        x, h = s["x"].to(f8), None
        if "delta" in s:
            h = x + s["delta"].to(f8)
            x = h.to(TORCH[case["x"]]).to(f8)      # the norm is of h as it is stored
        if case["op"] == "norm":
            x = x * s["w"].to(f8) / torch.sqrt((x * x).sum(1, keepdim=True) / case["d"] + EPS)
        step = torch.stack([t.abs().max(1).values for t in x.split(128, 1)]) / 448
        # values at the border between two codes go by the last bits of fp32: no value is given for them
        out = {"codes": None, "scale": step}
        if case["op"] == "norm":
            out["h"] = h
        return out
    ql, kl = _lengths(case)
    page, hd, kv, nh = case["page"], case["hd"], case["n_kv"], case["n_head"]
    G = nh // kv
    starts = s["q_start"].tolist()
    if case["op"] == "select":
        means = s["means"].to(f8)
        for i, (first, last) in enumerate(_completed(case)):
            if last > first:
                at = s["table"][i, first:last].long()
                means[at] = _exact_pages(case, s, "k", at).mean(2)
        return {"means": means, "sel": None}
    out = torch.zeros(s["n_rows"], nh, hd, dtype=f8, device=DEV)
    lists = s["sel"].cpu().tolist()
    head = torch.arange(kv, device=DEV)[:, None]
    for i in range(case["n_seq"]):
        need = sorted({b for r in range(starts[i], starts[i + 1]) for one in lists[r] for b in one if b >= 0})
        where = {b: j for j, b in enumerate(need)}
        at = s["table"][i][torch.tensor(need, device=DEV)].long()
        K, V = (_exact_pages(case, s, w, at).transpose(0, 1) for w in ("k", "v"))     # [kv, pages, page, hd]
        for j in range(ql[i]):
            r, pos = starts[i] + j, kl[i] - ql[i] + j
            L = max(sum(b >= 0 for b in one) for one in lists[r])    # the same for every head of a row
            idx = torch.tensor([[where[b] for b in one[:L]] for one in lists[r]], device=DEV)
            k, v = K[head, idx].reshape(kv, L * page, hd), V[head, idx].reshape(kv, L * page, hd)
            n = (L - 1) * page + pos % page + 1                      # the row's own block is the last
            z = torch.matmul(s["q"][r].to(f8).view(kv, G, hd), k[:, :n].transpose(1, 2).contiguous()) / math.sqrt(hd)
            out[r] = torch.matmul(torch.softmax(z, -1), v[:, :n].contiguous()).view(nh, hd)
    return out.view(s["n_rows"], nh * hd)


def _exact_pages(case, s, w, pages):
    """K or V [pages, n_kv, page, hd] of some pages, in 64 bits."""
    kv, page, hd = case["n_kv"], case["page"], case["hd"]
    if case["cache"] != "q4":
        t = s[w + "_pool"].view(TORCH[case["cache"]]).view(-1, kv, page * hd)[pages].double()
        return t.view(-1, kv, page, hd) if w == "k" else t.view(-1, kv, page // 8, hd, 8).permute(0, 1, 2, 4, 3).reshape(-1, kv, page, hd)
    raw = s[w + "_pool"].view(-1, kv, page * hd * 5 // 8)[pages]
    code = raw[..., :page * hd // 2].contiguous().view(-1, kv, page * hd // 8, 4)
    # byte b of a word holds elements 2b' (b < 2) or 2b'+1 (b >= 2): low nibble, then high nibble
    lo, hi = code & 15, code >> 4
    e = [None] * 8
    for b in range(4):
        e[4 * (b % 2) + b // 2], e[4 * (b % 2) + 2 + b // 2] = lo[..., b], hi[..., b]
    n = torch.stack(e, -1).double()
    sc = raw[..., page * hd // 2:].contiguous().view(torch.float16).double()
    if w == "k":
        sc = sc.view(-1, kv, page, hd // 32, 2)
        d, m, n = sc[..., 0], sc[..., 1], n.view(-1, kv, page, hd)
    else:
        sc = sc.view(-1, kv, page // 8, hd // 32, 2, 8)
        d, m = (sc[..., j, :].transpose(-1, -2).reshape(-1, kv, page, hd // 32) for j in (0, 1))
        n = n.view(-1, kv, page // 8, hd, 8).transpose(-1, -2).reshape(-1, kv, page, hd)
    return (m.repeat_interleave(32, -1) + d.repeat_interleave(32, -1) * n).half().double()
