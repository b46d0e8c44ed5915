"""Serving operators: paged KV cache append and read-back, attention over the paged cache (16-bit or
4-bit pages, decode rows and prompts), residual + RMSNorm to int8 rows, and rows to int8.

Each case is one call (or the calls a program makes together) on device tensors.  Lengths of ragged
batches follow from the case alone; values, page numbers and weights from the seed.  Layouts and
formulas are those of include/x100_paged.h and include/x100_rows.h.

  python3 -c "import sys; sys.path.insert(0, 'perf'); import operators as o; print(o.listed())"
"""
import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"
TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i32": torch.int32}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "i32": 4}
# bit position of element e of 8 in a 32-bit word of 4-bit codes: even elements in the low half
SHIFT = [0, 16, 4, 20, 8, 24, 12, 28]
EPS, ROPE_BASE = 1e-6, 1e6


def _case(name, **kw):
    return dict({"name": name}, **kw)


HEADS = dict(n_head=32, n_kv=4, hd=128)     # 32 query heads on 4 KV heads of 128


def listed():
    return [
        # one user, a short chat: the attention of one new token
        _case("decode 1x1024 bf16", op="attn", n_seq=1, q=1, kv=1024, page=64, act="bf16", cache="bf16", **HEADS),
        # a server's decode step: 64 sequences of different lengths
        _case("decode 64x4096 f16", op="attn", n_seq=64, q=1, kv=4096, page=16, act="f16", cache="f16", **HEADS),
        # long contexts kept in 4 bits, one token each
        _case("decode 16x60001 q4", op="attn", n_seq=16, q=1, kv=60001, page=64, act="bf16", cache="q4", **HEADS),
        # prompts of several users in one batch, nothing cached before them
        _case("prompt 4x4000 bf16", op="attn", n_seq=4, q=4000, kv=4000, page=64, act="bf16", cache="bf16", **HEADS),
        # pieces of prompts behind long cached prefixes, in 4 bits, heads of 64
        _case("chunk 3x509 on 16384 q4", op="attn", n_seq=3, q=509, kv=16384, page=32, act="f16", cache="q4",
              n_head=32, n_kv=8, hd=64),
        # one decode step's rows: a token per sequence, from fp32 projections, head norms
        _case("append 64 rows f32 to bf16", op="append", n_seq=64, q=1, kv=500, page=64, act="bf16", cache="bf16",
              src="f32", norm=True, **HEADS),
        # the same for few sequences into 4 bits, read back
        _case("append 8 rows bf16 to q4", op="append", n_seq=8, q=1, kv=4096, page=64, act="bf16", cache="q4",
              src="bf16", norm=True, **HEADS),
        # prompts straight from the int8 GEMM's int32 sums, into 4 bits, read back
        _case("append 6x2011 rows i32 to q4", op="append", n_seq=6, q=2011, kv=2100, page=64, act="f16", cache="q4",
              src="i32", norm=True, **HEADS),
        # residual and norm in front of the projections: a decode step, and a prompt after the int8 GEMM of Wo
        _case("norm 64x2048 f32", op="norm", rows=64, d=2048, x="f32", delta="f32"),
        _case("norm 16381x2048 bf16 i32", op="norm", rows=16381, d=2048, x="bf16", delta="i32"),
        # the attention's output in front of Wo's int8 GEMM
        _case("quant 16x4096 bf16", op="quant", rows=16, d=4096, x="bf16"),
        _case("quant 16384x4096 f16", op="quant", rows=16384, d=4096, x="f16"),
    ]


def _logint(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["decode", "decode", "prompt", "prompt", "append", "append", "norm", "quant"])
    if op in ("norm", "quant"):
        d = rng.choice([_logint(rng, 64, 8192), 16 * _logint(rng, 16, 512), 512, 1024, 2048, 4096])
        rows = _logint(rng, 1, max(1, min(16000, 32000000 // d)))
        c = dict(op=op, rows=rows, d=d, x=rng.choice(["f32", "f16", "bf16"]))
        if op == "norm":
            c["delta"] = rng.choice(["f32", "f16", "bf16", "i32", "none"])
        return c
    hd = rng.choice([64, 128, 128])
    n_kv = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 3, 4, 5, 8, 8, 16]) if n_kv <= 4 else rng.choice([1, 2, 4])
    act = rng.choice(["f16", "bf16"])
    c = dict(n_head=n_kv * group, n_kv=n_kv, hd=hd, page=rng.choice([16, 32, 64, 128, 256]), act=act,
             cache=rng.choice([act, "q4"]))
    if op == "decode":
        kv = _logint(rng, 1, 60000)
        most = max(1, min(256, 900000 * 512 // (kv * n_kv * hd)))
        return dict(c, op="attn", n_seq=_logint(rng, 1, most), q=rng.choice([1, 1, 1, 2, 4]), kv=max(4, kv))
    if op == "prompt":
        q = _logint(rng, 5, 4000)
        kv = q + rng.choice([0, 0, _logint(rng, 1, 12000)])
        most = max(1, min(24, int(1.5e9 / (q * kv * c["n_head"]))))
        if q * kv * c["n_head"] > 1.5e9:
            kv = q
        return dict(c, op="attn", n_seq=_logint(rng, 1, most), q=q, kv=kv)
    q = rng.choice([1, _logint(rng, 1, 2500)])
    width = (c["n_head"] + 2 * n_kv) * hd
    n_seq = _logint(rng, 1, max(1, min(192, 50000000 // (q * width))))
    return dict(c, op="append", n_seq=n_seq, q=q, kv=q + _logint(rng, 1, 2000),
                src=rng.choice(["f32", "f16", "bf16", "i32"]), norm=rng.choice([True, False]))


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


def _row_types(case):
    return case["src"] if case["op"] == "append" else case["act"]


def _pool_bytes(case, n_pages):
    per = case["hd"] * 2 if case["cache"] != "q4" else case["hd"] * 5 // 8
    return n_pages * case["n_kv"] * case["page"] * per


def work(case):
    if case["op"] in ("norm", "quant"):
        n, s = case["rows"] * case["d"], SIZE[case["x"]]
        if case["op"] == "quant":
            return {"bytes": n * (s + 1) + 4 * case["rows"], "flops": 3 * n}
        t = case["delta"]
        b = n * (s + 1 + (0 if t == "none" else SIZE[t] + s)) + 4 * case["rows"] + 4 * case["d"]
        return {"bytes": b, "flops": 6 * n}
    ql, kl = _lengths(case)
    per = case["hd"] * (2.0 if case["cache"] != "q4" else 0.625)     # bytes of a K (or V) head row
    rows, hd = sum(ql), case["hd"]
    if case["op"] == "append":
        width = (case["n_head"] + 2 * case["n_kv"]) * hd
        b = rows * (width * SIZE[case["src"]] + case["n_head"] * hd * 2 + 2 * case["n_kv"] * per)
        if case["cache"] == "q4":                                    # read back in 16 bits
            b += rows * 2 * case["n_kv"] * (per + hd * 2)
        return {"bytes": b, "flops": 8 * rows * width}
    seen = sum(a * (k - a) + a * (a + 1) // 2 for a, k in zip(ql, kl))
    return {"bytes": sum(kl) * case["n_kv"] * 2 * per + 2 * rows * case["n_head"] * hd * 2,
            "flops": 4 * seen * case["n_head"] * hd}


# ---- the 4-bit format: groups of 32 along the head, value = fp16(m + d * n) -----------------------

def _q4(x):
    """x [..., hd] fp32 -> codes [..., hd] (int32), d and m [..., hd/32] (fp16)."""
    g = x.reshape(*x.shape[:-1], -1, 32)
    lo, hi = g.amin(-1), g.amax(-1)
    d, m = ((hi - lo) / 15.0).half(), lo.half()
    bad = ~(torch.isfinite(g).all(-1) & torch.isfinite(d) & torch.isfinite(m))
    df = d.float()
    inv = torch.where(df > 0, 1.0 / df, torch.zeros_like(df))
    n = torch.round((g - m.float()[..., None]) * inv[..., None]).clamp(0, 15)
    n = torch.where(bad[..., None], torch.zeros_like(n), n).to(torch.int32)
    nan = torch.full_like(d, float("nan"))
    return n.reshape(x.shape), torch.where(bad, nan, d), torch.where(bad, nan, m)


def _q4_values(n, d, m):
    """codes [..., hd], d and m [..., hd/32] -> fp16 values (one rounding: d n + m is formed in fp64)."""
    g = n.reshape(*n.shape[:-1], -1, 32).double()
    return (g * d.double()[..., None] + m.double()[..., None]).half().reshape(n.shape)


def _views(case, pool, which):
    """The pool's parts: 16 bits one tensor; 4 bits (codes, scales)."""
    kv, page, hd = case["n_kv"], case["page"], case["hd"]
    if case["cache"] != "q4":
        t = pool.view(TORCH[case["cache"]])
        return t.view(-1, kv, page, hd) if which == "k" else t.view(-1, kv, page // 8, hd, 8)
    b = pool.view(-1, kv, page * hd * 5 // 8)
    codes, scales = b[..., :page * hd // 2].view(torch.int32), b[..., page * hd // 2:].view(torch.float16)
    return codes, scales


def _gather(case, pool, which, table):
    """Values of the pages in table [n_seq, n]: [n_seq, n_kv, n * page, hd] (fp32)."""
    kv, page, hd = case["n_kv"], case["page"], case["hd"]
    S, n = table.shape
    if case["cache"] != "q4":
        t = _views(case, pool, which)[table]                 # [S, n, kv, ...]
        if which == "v":
            t = t.transpose(-1, -2)                          # [S, n, kv, page/8, 8, hd]
        return t.float().reshape(S, n, kv, page, hd).transpose(1, 2).reshape(S, kv, n * page, hd)
    codes, scales = _views(case, pool, which)
    sh = torch.tensor(SHIFT, device=pool.device, dtype=torch.int32)
    c, s = codes[table], scales[table]
    c = (c[..., None] >> sh) & 15                            # [S, n, kv, words, 8]
    if which == "k":
        c = c.reshape(S, n, kv, page, hd)
        d, m = s.reshape(S, n, kv, page, hd // 32, 2).unbind(-1)
    else:
        c = c.reshape(S, n, kv, page // 8, hd, 8).transpose(-1, -2).reshape(S, n, kv, page, hd)
        s = s.reshape(S, n, kv, page // 8, hd // 32, 2, 8)
        d, m = (s[..., i, :].transpose(-1, -2).reshape(S, n, kv, page, hd // 32) for i in (0, 1))
    g = c.reshape(S, n, kv, page, hd // 32, 32).float()
    # d n + m in fp32: d n is exact (11 + 4 bits); the sum rounds once more before fp16 only where m
    # and d n are far apart
    v = (g * d.float()[..., None] + m.float()[..., None]).half().float()
    return v.reshape(S, n, kv, page, hd).transpose(1, 2).reshape(S, kv, n * page, hd)


# ---- what a program has in hand -------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed * 1000003 + 17)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    def rows(n, width, kind):
        """n rows of a type; int32: what an int8 GEMM leaves, with its row and column scales."""
        if kind != "i32":
            return normal(n, width).to(TORCH[kind]), None, None
        t = (normal(n, width) * 30000).round().to(torch.int32)
        rs = (0.5 + torch.rand(n, generator=g, device=DEV)) / 300
        cs = (0.5 + torch.rand(width, generator=g, device=DEV)) / 100
        return t, rs, cs

    s = {"case": case}
    if case["op"] in ("norm", "quant"):
        n, d = case["rows"], case["d"]
        s["x"] = (normal(n, d) * (0.5 + 4 * torch.rand(n, 1, generator=g, device=DEV))).to(TORCH[case["x"]])
        s["q"] = torch.empty(n, d, dtype=torch.int8, device=DEV)
        s["scale"] = torch.empty(n, device=DEV)
        if case["op"] == "norm":
            s["w"] = 1 + 0.2 * normal(d)
            if case["delta"] != "none":
                s["delta"], s["rs"], s["cs"] = rows(n, d, case["delta"])
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
        for w in ("k", "v"):
            vals = n_pages * kv * page * hd
            if case["cache"] != "q4":
                pool = torch.empty(vals, dtype=TORCH[case["cache"]], device=DEV).normal_(generator=g)
            else:     # random codes with the scales that normal values get: 15 steps over about 4 deviations
                pool = torch.empty(n_pages * kv, page * hd * 5 // 8, dtype=torch.uint8, device=DEV)
                pool[:, :page * hd // 2] = torch.randint(0, 256, (n_pages * kv, page * hd // 2), generator=g,
                                                         device=DEV, dtype=torch.uint8)
                d = 0.25 + 0.1 * torch.rand(n_pages * kv * page * hd // 32, generator=g, device=DEV)
                m = -7.5 * d + 0.3 * normal(d.numel())
                if w == "k":
                    sc = torch.stack([d, m], -1)
                else:
                    sc = torch.stack([d.view(-1, 8), m.view(-1, 8)], 1)
                pool[:, page * hd // 2:] = sc.half().reshape(n_pages * kv, -1).view(torch.uint8)
            s[w + "_pool"] = pool.view(torch.uint8).reshape(-1)
        if case["op"] == "attn":
            # scores of about 1.5 deviations, as heads with normalised queries and keys have them
            s["q"] = (1.5 * normal(n, nh * hd)).to(TORCH[case["act"]])
            s["out"] = torch.empty_like(s["q"])
        else:
            s["src"], s["rs"], s["cs"] = rows(n, (nh + 2 * kv) * hd, case["src"])
            s["qn"], s["kn"] = (1 + 0.2 * normal(hd), 1 + 0.2 * normal(hd)) if case["norm"] else (None, None)
            ang = torch.arange(case["kv"], device=DEV, dtype=torch.float64)[:, None] * \
                ROPE_BASE ** (-torch.arange(0, hd, 2, device=DEV, dtype=torch.float64) / hd)
            s["rope"] = torch.stack([ang.cos(), ang.sin()], -1).float().contiguous()
            s["q_out"] = torch.empty(n, nh * hd, dtype=TORCH[case["act"]], device=DEV)
            if case["cache"] == "q4":
                s["k_rows"] = torch.empty(n, kv * hd, dtype=TORCH[case["act"]], device=DEV)
                s["v_rows"] = torch.empty_like(s["k_rows"])
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
    T = {"f32": x.T_F32, "f16": x.T_F16, "bf16": x.T_BF16, "i32": x.T_I32, "q4": x.KV_Q4}
    p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    if case["op"] in ("norm", "quant"):
        s["rx"] = x.Rows(T[case["x"]], p(s["x"]), case["d"], None, None)
        s["rd"] = x.Rows(T[case["delta"]], p(s["delta"]), case["d"], p(s["rs"]), p(s["cs"])) if "delta" in s else None
        return
    s["cfg"] = x.KvCfg(case["n_head"], case["n_kv"], case["hd"], case["page"], s["n_pages"], T[case["act"]],
                       T[case["cache"]])
    s["batch"] = x.KvBatch(case["n_seq"], s["n_rows"], case["q"], case["kv"], s["table"].shape[1], p(s["q_start"]),
                           p(s["kv_len"]), p(s["table"]))
    if case["op"] == "attn":
        n = x.attn_paged_workspace_bytes(s["cfg"], s["batch"])
        s["ws"] = torch.empty(max(n, 256), dtype=torch.uint8, device=DEV)
        return
    nh, kv, hd = case["n_head"], case["n_kv"], case["hd"]
    width, size = (nh + 2 * kv) * hd, SIZE[case["src"]]
    r = []
    for col in (0, nh * hd, (nh + kv) * hd):
        cs = None if s["cs"] is None else p(s["cs"]) + 4 * col
        r.append(x.Rows(T[case["src"]], p(s["src"]) + col * size, width, p(s["rs"]), cs))
    s["rows"] = x.KvRows(r[0], r[1], r[2], p(s["qn"]), p(s["kn"]), EPS, p(s["rope"]), case["kv"])


def _run_own(s):
    x, case = s["lib"], s["case"]
    stream = torch.cuda.current_stream().cuda_stream
    if case["op"] == "quant":
        x.quant_i8(case["rows"], case["d"], s["rx"], s["q"].data_ptr(), s["scale"].data_ptr(), stream)
        return {"values": s["q"] * s["scale"][:, None], "scale": s["scale"]}
    if case["op"] == "norm":
        h = s.get("h")
        x.add_rmsnorm_i8(case["rows"], case["d"], s["rx"], s["rd"], s["w"].data_ptr(), EPS,
                         None if h is None else h.data_ptr(), case["d"], s["q"].data_ptr(), s["scale"].data_ptr(),
                         stream)
        return {"values": s["q"] * s["scale"][:, None], "scale": s["scale"], "h": h}
    k, v = s["k_pool"].data_ptr(), s["v_pool"].data_ptr()
    if case["op"] == "attn":
        w = case["n_head"] * case["hd"]
        x.attn_paged_ws(s["cfg"], s["batch"], s["q"].data_ptr(), w, k, v, case["hd"] ** -0.5, s["out"].data_ptr(), w,
                        s["ws"].data_ptr(), s["ws"].numel(), stream)
        return s["out"]
    x.kv_append(s["cfg"], s["batch"], s["rows"], k, v, s["q_out"].data_ptr(), stream)
    if case["cache"] != "q4":
        return {"q": s["q_out"], "k": s["k_pool"].view(TORCH[case["cache"]]),
                "v": s["v_pool"].view(TORCH[case["cache"]])}
    x.kv_read(s["cfg"], s["batch"], k, v, s["k_rows"].data_ptr(), s["v_rows"].data_ptr(), stream)
    return {"q": s["q_out"], "k": s["k_rows"], "v": s["v_rows"]}


# ---- the plain forms ------------------------------------------------------------------------------

def _real(t, rs, cs):
    return t.float() if rs is None else t.float() * rs[:, None] * cs


def _codes(t):
    """Rows t (fp32) -> (codes as fp32, amax): code = rint(t * (127 / amax)); a row that is all (nearly)
    zero has codes 0, one that holds a value that is not finite amax NaN."""
    amax = t.abs().amax(1)
    ok = torch.isfinite(t).all(1)
    some = ok & (amax >= 2.0 ** -100)
    inv = torch.where(some, 127.0 / amax, torch.zeros_like(amax))
    c = torch.round(t * inv[:, None])
    c = torch.where(some[:, None], c, torch.zeros_like(c))
    amax = torch.where(some, amax, torch.where(ok, torch.zeros_like(amax), torch.full_like(amax, float("nan"))))
    return c, amax


def _positions(s):
    """seq and pos of every row."""
    n = s["n_rows"]
    r = torch.arange(n, device=DEV)
    seq = torch.searchsorted(s["q_start"][1:].long(), r, right=True)
    pos = s["kv_len"].long()[seq] - s["q_start"].long()[seq + 1] + r
    return r, seq, pos


def _run_plain(s):
    case = s["case"]
    if case["op"] == "quant":
        c, amax = _codes(s["x"].float())
        scale = amax / 127.0
        return {"values": c * scale[:, None], "scale": scale}
    if case["op"] == "norm":
        x, h = s["x"].float(), None
        if "delta" in s:
            h = (x + _real(s["delta"], s["rs"], s["cs"])).to(TORCH[case["x"]])
            x = h.float()
        r = 1.0 / torch.sqrt(x.square().mean(1) + EPS)
        c, amax = _codes(x * s["w"])
        scale = amax * r / 127.0
        return {"values": c * scale[:, None], "scale": scale, "h": h}
    page, hd, kv, nh = case["page"], case["hd"], case["n_kv"], case["n_head"]
    r, seq, pos = _positions(s)
    if case["op"] == "attn":
        S, q = case["n_seq"], case["q"]
        i = r - s["q_start"].long()[seq]
        K, V = (_gather(case, s[w + "_pool"], w, s["table"].long()) for w in ("k", "v"))
        Q = torch.zeros(S, q, nh * hd, device=DEV)
        Q[seq, i] = s["q"].float()
        P = torch.full((S, q), -1, device=DEV, dtype=torch.long)
        P[seq, i] = pos
        Q = Q.view(S, q, kv, nh // kv, hd).permute(0, 2, 3, 1, 4).reshape(S, kv, nh // kv * q, hd)
        sc = torch.matmul(Q, K.transpose(-1, -2)) * hd ** -0.5
        sc = sc.view(S, kv, nh // kv, q, -1)
        far = torch.arange(K.shape[2], device=DEV)[None, None, :] > P[:, :, None]
        sc.masked_fill_(far[:, None, None], float("-inf"))
        top = sc.amax(-1, keepdim=True)
        sc.sub_(torch.where(top == float("-inf"), torch.zeros_like(top), top)).exp_()
        den = sc.sum(-1, keepdim=True)
        o = torch.matmul(sc.view(S, kv, nh // kv * q, -1), V).view(S, kv, nh // kv, q, hd)
        o = torch.where(den > 0, o / den, torch.zeros_like(o))
        return o.permute(0, 3, 1, 2, 4).reshape(S, q, nh * hd)[seq, i].to(TORCH[case["act"]])
    n = s["n_rows"]
    x = _real(s["src"], s["rs"], s["cs"]).view(n, nh + 2 * kv, hd)
    cs, sn = s["rope"][pos].unbind(-1)

    def turned(t, w):
        if w is not None:
            t = t * (1.0 / torch.sqrt(t.square().mean(-1, keepdim=True) + EPS)) * w
        a, b = t[..., :hd // 2], t[..., hd // 2:]
        c, d = cs[:, None], sn[:, None]
        return torch.cat([a * c - b * d, a * d + b * c], -1)

    q_out = turned(x[:, :nh], s["qn"]).to(TORCH[case["act"]]).view(n, nh * hd)
    k, v = turned(x[:, nh:nh + kv], s["kn"]), x[:, nh + kv:]
    at, off = s["table"].long()[seq, pos // page], pos % page
    if case["cache"] != "q4":
        kp, vp = _views(case, s["k_pool"], "k"), _views(case, s["v_pool"], "v")
        kp[at, :, off] = k.to(kp.dtype)
        vp[at, :, off // 8, :, off % 8] = v.to(vp.dtype)
        return {"q": q_out, "k": s["k_pool"].view(kp.dtype), "v": s["v_pool"].view(vp.dtype)}
    sh = torch.tensor(SHIFT, device=DEV, dtype=torch.int32)
    head = torch.arange(kv, device=DEV)
    # keys: a word holds 8 elements of one row
    c, d, m = _q4(k)
    words = (c.view(n, kv, hd // 8, 8) << sh).sum(-1, dtype=torch.int64).to(torch.int32)
    kc, ks = _views(case, s["k_pool"], "k")
    kc.view(-1, kv, page, hd // 8)[at, :, off] = words
    ks.view(-1, kv, page, hd // 32, 2)[at, :, off] = torch.stack([d, m], -1)
    k_rows = _q4_values(c, d, m)
    # values: a word holds 8 positions of one element, so a row changes 4 bits of every word
    c, d, m = _q4(v)
    vc, vs = _views(case, s["v_pool"], "v")
    blk, at1, bit = off // 8, at[:, None], sh[off % 8][:, None, None]
    w = vc.view(-1, kv, page // 8, hd)
    here = (at1, head[None], blk[:, None])
    w.index_put_(here, (c - ((w[here] >> bit) & 15)) << bit, accumulate=True)
    vs.view(-1, kv, page // 8, hd // 32, 2, 8)[at, :, blk, :, :, off % 8] = torch.stack([d, m], -1)
    act = TORCH[case["act"]]
    return {"q": q_out, "k": k_rows.to(act).view(n, kv * hd), "v": _q4_values(c, d, m).to(act).view(n, kv * hd)}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the definitions in 64 bits -------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    f8 = torch.float64
    if case["op"] in ("norm", "quant"):
        if case["rows"] * case["d"] > 1 << 28:
            return None
        x, h = s["x"].to(f8), None
        if "delta" in s:
            t = s["delta"].to(f8)
            if case["delta"] == "i32":
                t = torch.einsum("ij,i,j->ij", t, s["rs"].to(f8), s["cs"].to(f8))
            h = x + t
            x = h.to(TORCH[case["x"]]).to(f8)      # the norm is of h as it is stored
        if case["op"] == "norm":
            x = x / torch.sqrt((x * x).sum(1, keepdim=True) / case["d"] + EPS) * s["w"].to(f8)
        step = x.abs().max(1, keepdim=True).values / 127
        # values at the border between two codes go by the last bits of fp32: no value is given for them
        out = {"values": None, "scale": step[:, 0]}
        if case["op"] == "norm":
            out["h"] = h
        return out
    ql, kl = _lengths(case)
    page, hd, kv, nh = case["page"], case["hd"], case["n_kv"], case["n_head"]
    G = nh // kv
    starts = s["q_start"].tolist()
    if case["op"] == "attn":
        out = torch.zeros(s["n_rows"], nh, hd, dtype=f8, device=DEV)
        for i in range(case["n_seq"]):
            L, n, r0 = kl[i], ql[i], starts[i]
            pages = s["table"][i].long()[:-(-L // page)]
            K, V = _exact_pages(case, s, pages)
            q = s["q"][r0:r0 + n].to(f8).view(n, nh, hd)
            last = torch.arange(L - n, L, device=DEV)
            hidden = torch.arange(L, device=DEV)[None, :] > last[:, None]
            for h in range(kv):
                z = q[:, h * G:(h + 1) * G].permute(1, 0, 2).reshape(G * n, hd) @ K[h, :L].T / math.sqrt(hd)
                z = z.view(G, n, L).masked_fill(hidden, float("-inf"))
                z = torch.softmax(z, -1)
                out[r0:r0 + n, h * G:(h + 1) * G] = (z.view(G * n, L) @ V[h, :L]).view(G, n, hd).permute(1, 0, 2)
        return out.view(s["n_rows"], nh * hd)
    x = s["src"].to(f8)
    if case["src"] == "i32":
        x = x * torch.outer(s["rs"].to(f8), s["cs"].to(f8))
    pos = torch.cat([torch.arange(k - a, k, device=DEV) for a, k in zip(ql, kl)])
    z = torch.polar(torch.ones((), dtype=f8, device=DEV),
                    pos[:, None].to(f8) / ROPE_BASE ** (torch.arange(hd // 2, device=DEV, dtype=f8) * 2 / hd))
    parts = []
    for part, w in ((x[:, :nh * hd], s["qn"]), (x[:, nh * hd:(nh + kv) * hd], s["kn"])):
        t = part.reshape(len(pos), -1, hd)
        if w is not None:
            t = t * torch.rsqrt(t.pow(2).mean(-1, keepdim=True) + EPS) * w.to(f8)
        c = torch.complex(t[..., :hd // 2], t[..., hd // 2:]) * z[:, None, :]
        parts.append(torch.cat([c.real, c.imag], -1).reshape(len(pos), -1))
    q, k = parts
    v = x[:, (nh + kv) * hd:]
    if case["cache"] != "q4":
        out = {"q": q}
        seq = torch.cat([torch.full((a,), i, device=DEV) for i, a in enumerate(ql)])
        at = s["table"].long()[seq, pos // page]
        for name, t in (("k", k), ("v", v)):
            pool = s[name + "_pool"].view(TORCH[case["cache"]]).to(f8)
            t = t.reshape(len(pos), kv, hd)
            for h in range(kv):
                base = (at * kv + h) * page * hd
                o = pos % page
                el = torch.arange(hd, device=DEV)
                if name == "k":
                    pool[(base + o * hd)[:, None] + el] = t[:, h]
                else:
                    pool[(base + o // 8 * 8 * hd + o % 8)[:, None] + 8 * el] = t[:, h]
            out[name] = pool
        return out
    out = {"q": q}
    for name, t in (("k", k), ("v", v)):
        g = t.reshape(len(pos), -1, 32)
        lo, hi = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
        d, m = ((hi - lo) / 15).half().to(f8), lo.half().to(f8)
        n = ((g - m) / d).round().clamp(0, 15)
        out[name] = (m + d * n).half().to(f8).reshape(len(pos), kv * hd)
    return out


def _exact_pages(case, s, pages):
    """K and V [n_kv, positions, hd] of a sequence's pages, in 64 bits."""
    kv, page, hd = case["n_kv"], case["page"], case["hd"]
    got = []
    for w in ("k", "v"):
        if case["cache"] != "q4":
            t = s[w + "_pool"].view(TORCH[case["cache"]]).view(-1, kv, page * hd)[pages].double()
            t = t.view(-1, kv, page, hd) if w == "k" else t.view(-1, kv, page // 8, hd, 8).permute(0, 1, 2, 4, 3)
        else:
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
            d, m = d.repeat_interleave(32, -1), m.repeat_interleave(32, -1)
            t = (m + d * n).half().double()
        got.append(t.reshape(-1, kv, page, hd).transpose(0, 1).reshape(kv, -1, hd))
    return got
