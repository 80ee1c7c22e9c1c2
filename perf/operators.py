"""Measured cases of the 8-bit K/V cache path and of the token log probabilities.

Four operators, each in a plain form (elementary torch operations) and as the call a user makes of the framework:

  * ``store``: one pass over projected q / k / v rows (per-head RMS norms of q and k, position rotation, the paged cache
    write in bf16, e4m3 or int8), then the stored rows read back, as a chunked prefill does that attends to the values
    the cache holds;
  * ``load``: rows of a long-lived 8-bit cache read back by slot (a prefix handed to a bf16 path);
  * ``attend``: one to a few new tokens per request attend over the paged 8-bit cache;
  * ``logprobs``: log probability, rank, entropy and best alternatives of given tokens.

An 8-bit cache row is one (token, K/V head): 128 codes and one power-of-two exponent e, the smallest e in [-40, 40]
with max|x| <= top * 2^e (top = 448 for e4m3, 127 for int8); code = round-half-even(x * 2^-e) on the code's grid.
"""
from __future__ import annotations

import math

import torch

own = False

D = 128            # head dimension
PAGE = 16          # tokens of a cache page
THETA = 10000.0    # base of the rotation frequencies
E_MIN, E_MAX = -40, 40
TOP = {"e4m3": 448.0, "int8": 127.0}
CODE = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------- cases
def _store(name, m, fmt, *, norm=True, half=False, rd=64, mrope=False, nq=16, nkv=8, far=8192):
    return {"name": name, "kind": "store", "m": m, "fmt": fmt, "norm": norm, "half": half, "rd": rd, "mrope": mrope,
            "nq": nq, "nkv": nkv, "far": far}


def _load(name, n, fmt, *, pages, nkv=8):
    return {"name": name, "kind": "load", "n": n, "fmt": fmt, "pages": pages, "nkv": nkv}


def _attend(name, bs, lo, hi, fmt, *, K=1, draft=0, nq=16, nkv=8):
    return {"name": name, "kind": "attend", "bs": bs, "lo": lo, "hi": hi, "fmt": fmt, "K": K, "draft": draft,
            "nq": nq, "nkv": nkv}


def _logprobs(name, rows, vocab, dtype, n_top, *, warm=False, masked=0.0):
    return {"name": name, "kind": "logprobs", "rows": rows, "vocab": vocab, "dtype": dtype, "n_top": n_top,
            "warm": warm, "masked": masked}


def listed():
    return [
        # one decode token of one request: latency only
        _store("store_1", 1, "int8"),
        # the verify rows of 64 requests at B = 16, multimodal positions, e4m3, no head norms (this decoder has none)
        _store("store_1088", 1088, "e4m3", norm=False, mrope=True),
        # a prefill of 16 requests of 1,031 tokens, head norms, the half-split rotation of the whole head
        _store("store_16496", 16496, "int8", half=True, rd=128, far=1031),
        # one request's prefix (256 image rows + 32 prompt rows + a ragged rest) handed to a bf16 path
        _load("load_301", 301, "e4m3", pages=4096),
        # 16 full-page requests of 4,160 tokens
        _load("load_66560", 66560, "int8", pages=4160),
        # one new token of one request behind a 2,738-token prefix: the batch-1 decode
        _attend("attend_1x2738", 1, 2738, 2738, "e4m3"),
        # one new token of 64 requests whose lengths spread over the serving mix's range
        _attend("attend_64x288_4128", 64, 288, 4128, "int8"),
        # one long document: the only parallelism is the cache's length
        _attend("attend_1x131071", 1, 131071, 131071, "e4m3"),
        # the verify rows [a0, d1..d16] of 64 requests, causal
        _attend("attend_64x17rows", 64, 288, 4128, "int8", K=17),
        # the token just drawn, its rank and 5 alternatives
        _logprobs("logprobs_1", 1, 59392, "fp32", 5),
        # a decode step of 64 requests with bf16 logits at a temperature
        _logprobs("logprobs_64", 64, 59392, "bf16", 20, warm=True),
        # every verify row of 64 requests at B = 16, grammar-masked logits
        _logprobs("logprobs_1088", 1088, 59392, "fp32", 20, masked=0.25),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["store", "load", "attend", "attend", "logprobs"])
    heads = rng.choice([(16, 8), (16, 8), (16, 2), (6, 6), (32, 8), (12, 4), (5, 1)])
    if kind == "store":
        half = rng.random() < 0.5
        rd = rng.choice([32, 64, 64, 96, 128])
        return _store(None, _log(rng, 1, 12000), rng.choice(["bf16", "e4m3", "int8"]), norm=rng.random() < 0.6,
                      half=half, rd=rd, mrope=rng.random() < 0.4, nq=min(heads[0], 16), nkv=heads[1],
                      far=_log(rng, 64, 262144))
    if kind == "load":
        n = _log(rng, 1, 66560)
        return _load(None, n, rng.choice(["bf16", "e4m3", "int8"]), pages=n // PAGE + 1 + _log(rng, 1, 2000),
                     nkv=min(8, heads[1]))
    if kind == "attend":
        bs = _log(rng, 1, 128)
        K = rng.choice([1, 1, 1, 1, 2, 3, 5, 9, 17])
        if heads[0] // heads[1] * K > 128:
            K = 1
        # no more rows x tokens than the 64 requests' verify rows: 64 x 17 x 2 x 2,208
        cap = 64 * 17 * 2 * 2208 // (bs * K * (heads[0] // heads[1]) * max(1, heads[1] // 8))
        hi = _log(rng, 1, max(1, min(131071, cap, 141000 // bs)))
        lo = hi if bs == 1 else max(0, int(hi * rng.uniform(0.0, 1.0)))
        return _attend(None, bs, lo, hi, rng.choice(["e4m3", "int8"]), K=K,
                       draft=rng.choice([0, 0, 1, 2]) if K > 1 else 0, nq=heads[0], nkv=heads[1])
    vocab = _log(rng, 1000, 131072)
    return _logprobs(None, _log(rng, 1, max(1, min(1088, 60_000_000 // vocab))), vocab, rng.choice(["fp32", "bf16"]),
                     rng.randint(1, 32), warm=rng.random() < 0.5, masked=rng.choice([0.0, 0.0, 0.25, 0.9]))


# ---------------------------------------------------------------------- the 8-bit rows, plain form
def _pow2(e):
    """2^e in 32 bits, exact, |e| < 127."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _exponent(amax, top):
    """Smallest e in [-40, 40] with amax <= top * 2^e."""
    m, k = torch.frexp(amax / top)                       # amax / top = m 2^k, 0.5 <= m < 1 (m = 0 for amax = 0)
    e = torch.where(m == 0.5, k - 1, k)
    # the division rounds: settle the border with exact products
    e = torch.where(amax == 0, torch.full_like(e, E_MIN), e).clamp(E_MIN - 1, E_MAX + 1).to(torch.int32)
    e = e + (top * _pow2(e) < amax).int() - (top * _pow2(e - 1) >= amax).int()
    return e.clamp(E_MIN, E_MAX)


def _codes(x, fmt):
    """Codes (as numbers in x's type) and exponents of rows x [..., 128]."""
    e = _exponent(x.abs().amax(-1), TOP[fmt])
    y = x * _pow2(-e)[..., None]
    if fmt == "int8":
        return torch.round(y).clamp(-127, 127), e
    k = (torch.frexp(y)[1] - 1).clamp_min(-6)            # |y| in [2^k, 2^(k+1)), or below the normal range
    step = _pow2(k - 3)
    return (torch.round(y / step) * step).clamp(-448, 448), e


def _values(codes, exps):
    return codes.float() * _pow2(exps)[..., None]


# ---------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=g, device="cuda", dtype=dtype)


def _new_cache(pages, nkv, fmt):
    k = torch.zeros((pages, nkv, PAGE, D), dtype=CODE[fmt], device="cuda")
    v = torch.zeros_like(k)
    if fmt == "bf16":
        return k, v, None, None
    ke = torch.zeros((pages, nkv, PAGE), dtype=torch.int8, device="cuda")
    return k, v, ke, torch.zeros_like(ke)


def _fill_cache(g, cache, fmt):
    """A cache as decoding leaves it: keys with a few loud channels, values whose size differs from token to token."""
    k, v, ke, ve = cache
    pages, nkv = k.shape[:2]
    loud = 1.0 + 7.0 * (torch.rand((1, nkv, 1, D), generator=g, device="cuda") < 0.04).float()
    for p0 in range(0, pages, 2048):
        n = min(2048, pages - p0)
        xk = (_randn(g, n, nkv, PAGE, D) * loud).bfloat16().float()
        xv = (_randn(g, n, nkv, PAGE, D) * torch.exp(_randn(g, n, nkv, PAGE, 1))).bfloat16().float()
        for x, c, e in ((xk, k, ke), (xv, v, ve)):
            if fmt == "bf16":
                c[p0: p0 + n] = x.bfloat16()
            else:
                q, ex = _codes(x, fmt)
                c[p0: p0 + n] = q.to(CODE[fmt])
                e[p0: p0 + n] = ex.to(torch.int8)


def _lens(case):
    """Tokens of each request's cache after this step's rows: evenly spread over [lo, hi], plus the K new rows."""
    bs, lo, hi = case["bs"], case["lo"], case["hi"]
    return [lo + (hi - lo) * i // max(1, bs - 1) + case["K"] for i in range(bs)]


def prepare(case, seed):
    g = _gen(seed)
    kind = case["kind"]
    s = {"case": case}
    if kind == "store":
        m, nq, nkv = case["m"], case["nq"], case["nkv"]
        width = (nq + 2 * nkv) * D
        x = _randn(g, m, width)
        x *= 1.0 + 5.0 * (torch.rand((1, width), generator=g, device="cuda") < 0.03).float()
        s["qkv"] = x.bfloat16()
        s["q_norm"] = (1.0 + 0.1 * _randn(g, D)).bfloat16() if case["norm"] else None
        s["k_norm"] = (1.0 + 0.1 * _randn(g, D)).bfloat16() if case["norm"] else None
        rd = case["rd"]
        s["inv_freq"] = (1.0 / THETA ** (torch.arange(0, rd, 2, device="cuda", dtype=torch.float64) / rd)).float()
        start = torch.randint(0, case["far"], (1,), generator=g, device="cuda")
        s["row_pos"] = s["row_pos3"] = None
        if case["mrope"]:
            t = torch.randint(0, case["far"], (m, 3), generator=g, device="cuda")
            s["row_pos3"] = t.to(torch.int32)
            a = rd // 8
            s["section"] = (a, (rd // 2 - a) // 2, rd // 2 - a - (rd // 2 - a) // 2)
        else:
            s["row_pos"] = ((start + torch.arange(m, device="cuda")) % case["far"]).to(torch.int32)
            s["section"] = None
        pages = m // PAGE + 17
        perm = torch.randperm(pages, generator=g, device="cuda")
        t = torch.arange(m, device="cuda") + 5
        s["slot"] = perm[t // PAGE] * PAGE + t % PAGE
        s["cache"] = _new_cache(pages, nkv, case["fmt"])
        s["q"] = torch.zeros((m, nq * D), dtype=torch.bfloat16, device="cuda")
        s["k"] = torch.zeros((m, nkv * D), dtype=torch.bfloat16, device="cuda")
        s["v"] = torch.zeros_like(s["k"])
    elif kind == "load":
        n, nkv, pages = case["n"], case["nkv"], case["pages"]
        s["cache"] = _new_cache(pages, nkv, case["fmt"])
        _fill_cache(g, s["cache"], case["fmt"])
        perm = torch.randperm(pages, generator=g, device="cuda")
        t = torch.arange(n, device="cuda")
        s["slot"] = perm[t // PAGE] * PAGE + t % PAGE
        s["k"] = torch.zeros((n, nkv * D), dtype=torch.bfloat16, device="cuda")
        s["v"] = torch.zeros_like(s["k"])
    elif kind == "attend":
        bs, K, nq, nkv = case["bs"], case["K"], case["nq"], case["nkv"]
        lens = _lens(case)
        per = (max(lens) + PAGE - 1) // PAGE
        used = [(n + PAGE - 1) // PAGE for n in lens]
        pages = sum(used) + 8
        s["cache"] = _new_cache(pages, nkv, case["fmt"])
        _fill_cache(g, s["cache"], case["fmt"])
        perm = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        table = torch.zeros((bs, per), dtype=torch.int32, device="cuda")
        o = 0
        for b in range(bs):
            table[b, : used[b]] = perm[o: o + used[b]]
            o += used[b]
        s["table"] = table
        s["seq"] = torch.tensor([n - K for n in lens], dtype=torch.int64, device="cuda")
        s["q"] = (_randn(g, bs * K, nq * D) * 0.5).bfloat16()
        s["out"] = torch.zeros((bs * K, nq * D), dtype=torch.bfloat16, device="cuda")
        s["lens"] = lens
    else:
        rows, vocab, n = case["rows"], case["vocab"], case["n_top"]
        x = _randn(g, rows, vocab) * 2.5
        hot = torch.randint(0, vocab, (rows, 8), generator=g, device="cuda")
        x.scatter_add_(1, hot, 5.0 + 10.0 * torch.rand((rows, 8), generator=g, device="cuda"))
        if case["masked"]:
            x.masked_fill_(torch.rand((1, vocab), generator=g, device="cuda") < case["masked"], float("-inf"))
            x[:, vocab // 2] = 1.0   # at least one token of each row stays
        s["logits"] = x.bfloat16() if case["dtype"] == "bf16" else x
        noise = -torch.log(-torch.log(torch.rand((rows, vocab), generator=g, device="cuda").clamp(1e-9, 1 - 1e-6)))
        s["ids"] = (s["logits"].float() + noise).argmax(1)
        s["temperature"] = (0.3 + 1.2 * torch.rand((rows,), generator=g, device="cuda")) if case["warm"] else None
        s["logprob"] = torch.zeros((rows,), device="cuda")
        s["entropy"] = torch.zeros((rows,), device="cuda")
        s["rank"] = torch.zeros((rows,), dtype=torch.int32, device="cuda")
        s["top"] = torch.zeros((rows, n), device="cuda")
        s["top_ids"] = torch.zeros((rows, n), dtype=torch.int32, device="cuda")
    if own:
        from gravityocr_b200 import _lib as L
        s["L"] = L
        s["status"] = torch.zeros((1,), dtype=torch.int32, device="cuda")
        if "cache" in s:
            s["handle"] = L.kv_cache(*s["cache"])
        if kind == "attend":
            a = (case["bs"], case["K"])
            s["split"] = L.kv8_attention_split(*a, max(s["lens"]), case["nq"], case["nkv"])
            need = L.kv8_attention_workspace_bytes(*a, case["nq"], case["nkv"], s["split"][1])
            s["ws"] = torch.zeros((need,), dtype=torch.uint8, device="cuda")
    return s


# ---------------------------------------------------------------------- plain forms
def _angles(s):
    """cos / sin [m, rotary_dim / 2] in 64 bits: a position times a frequency, exact to the last bit that matters."""
    f = s["inv_freq"].double()
    if s["row_pos3"] is None:
        a = s["row_pos"].double()[:, None] * f
    else:
        sec = torch.tensor(s["section"], device="cuda")
        axis = torch.repeat_interleave(torch.arange(3, device="cuda"), sec)
        a = s["row_pos3"].double()[:, axis] * f
    return torch.cos(a), torch.sin(a)


def _norm_rotate(x, w, eps, cos, sin, rd, half):
    """x [m, heads, 128] -> RMS norm times w (if given), then the rotation of the first rd elements, in x's type."""
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w.to(x.dtype)
    else:
        x = x.clone()
    c, s = cos.to(x.dtype)[:, None], sin.to(x.dtype)[:, None]
    if half:
        a, b = x[..., : rd // 2].clone(), x[..., rd // 2: rd].clone()
        x[..., : rd // 2], x[..., rd // 2: rd] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., 0:rd:2].clone(), x[..., 1:rd:2].clone()
        x[..., 0:rd:2], x[..., 1:rd:2] = a * c - b * s, b * c + a * s
    return x


EPS = 1e-5


def _plain_store(s):
    c = s["case"]
    m, nq, nkv, fmt = c["m"], c["nq"], c["nkv"], c["fmt"]
    x = s["qkv"].view(m, nq + 2 * nkv, D)
    cos, sin = _angles(s)
    q = _norm_rotate(x[:, :nq].float(), s["q_norm"], EPS, cos, sin, c["rd"], c["half"])
    # keys in 64 bits: a value next to a rounding border of the cache's grid has to fall on the right side of it
    k = _norm_rotate(x[:, nq: nq + nkv].double(), s["k_norm"], EPS, cos, sin, c["rd"], c["half"])
    v = x[:, nq + nkv:].float()
    page, off = s["slot"] // PAGE, s["slot"] % PAGE
    ck, cv, ke, ve = s["cache"]
    out = [q.bfloat16().view(m, nq * D)]
    for y, codes, exps in ((k, ck, ke), (v, cv, ve)):
        if fmt == "bf16":
            codes[page, :, off] = y.to(torch.bfloat16)
            got = codes[page, :, off]
        else:
            qc, e = _codes(y, fmt)
            codes[page, :, off] = qc.float().to(CODE[fmt])
            exps[page, :, off] = e.to(torch.int8)
            got = _values(codes[page, :, off], exps[page, :, off]).bfloat16()
        out.append(got.reshape(m, nkv * D))
    return out


def _plain_load(s):
    c = s["case"]
    page, off = s["slot"] // PAGE, s["slot"] % PAGE
    k, v, ke, ve = s["cache"]
    out = []
    for codes, exps in ((k, ke), (v, ve)):
        x = codes[page, :, off]
        if c["fmt"] != "bf16":
            x = _values(x, exps[page, :, off]).bfloat16()
        out.append(x.reshape(c["n"], c["nkv"] * D))
    return out


def _limits(case, seq):
    """Cache positions [0, limit) that each of the K window rows sees."""
    K = case["K"]
    if case["draft"] == 0:
        return [seq + j + 1 for j in range(K)]
    return [seq + 1 if (j == 0 and case["draft"] == 1) else seq + K for j in range(K)]


def _plain_attend(s):
    c = s["case"]
    bs, K, nq, nkv = c["bs"], c["K"], c["nq"], c["nkv"]
    G = nq // nkv
    ck, cv, ke, ve = s["cache"]
    out = torch.empty((bs * K, nq * D), dtype=torch.bfloat16, device="cuda")
    for b in range(bs):
        n = s["lens"][b]
        pages = s["table"][b, : (n + PAGE - 1) // PAGE].long()
        k = _values(ck[pages], ke[pages]).transpose(0, 1).reshape(nkv, -1, D)[:, :n]
        v = _values(cv[pages], ve[pages]).transpose(0, 1).reshape(nkv, -1, D)[:, :n]
        q = s["q"][b * K: (b + 1) * K].float().view(K, nkv, G, D).permute(1, 2, 0, 3).reshape(nkv, G * K, D)
        sc = (q @ k.transpose(1, 2) / math.sqrt(D)).view(nkv, G, K, n)
        if K > 1:
            lim = torch.tensor(_limits(c, n - K), device="cuda")
            sc = sc.masked_fill(torch.arange(n, device="cuda")[None, :] >= lim[:, None], float("-inf"))
        p = torch.exp(sc - sc.amax(-1, keepdim=True))
        o = (p.view(nkv, G * K, n) @ v).view(nkv, G, K, D) / p.sum(-1, keepdim=True)
        out[b * K: (b + 1) * K] = o.permute(2, 0, 1, 3).reshape(K, nq * D).bfloat16()
    return [out]


def _plain_logprobs(s):
    c = s["case"]
    raw = s["logits"].float()
    rows, vocab = raw.shape
    d = raw - raw.amax(1, keepdim=True)
    if s["temperature"] is not None:
        d = d / s["temperature"][:, None]
    e = torch.exp(d)
    total = e.sum(1, dtype=torch.float64)
    lse = torch.log(total)
    weighted = torch.where(e > 0, e * d, torch.zeros_like(d)).sum(1, dtype=torch.float64)
    entropy = lse - weighted / total
    mine = raw.gather(1, s["ids"][:, None])
    logprob = d.gather(1, s["ids"][:, None])[:, 0] - lse
    index = torch.arange(vocab, device="cuda")
    before = (raw > mine) | ((raw == mine) & (index[None, :] < s["ids"][:, None]))
    rank = before.sum(1) + 1
    # the best n, equal logits in the order of their ids: one integer key (ordered logit bits, descending id)
    bits = (raw + 0.0).view(torch.int32).long()
    key = torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF)) * (1 << 31) + (vocab - 1 - index)[None, :]
    best = torch.topk(key, c["n_top"], dim=1).values
    top_ids = vocab - 1 - (best & ((1 << 31) - 1))
    top = d.gather(1, top_ids) - lse[:, None]
    return [logprob.float(), entropy.float(), rank.to(torch.int32), top.float(), top_ids.to(torch.int32)]


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"store": _plain_store, "load": _plain_load, "attend": _plain_attend,
                "logprobs": _plain_logprobs}[c["kind"]](s)
    L = s["L"]
    if c["kind"] == "store":
        L.qk_norm_rope_write(s["qkv"], c["nq"], s["handle"], s["slot"], s["q"], s["inv_freq"], c["rd"],
                             row_pos=s["row_pos"], row_pos3=s["row_pos3"], mrope_section=s["section"],
                             rope_half=c["half"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS, status=s["status"])
        L.kv_read(s["handle"], s["slot"], s["k"], s["v"], status=s["status"])
        return [s["q"], s["k"], s["v"]]
    if c["kind"] == "load":
        L.kv_read(s["handle"], s["slot"], s["k"], s["v"], status=s["status"])
        return [s["k"], s["v"]]
    if c["kind"] == "attend":
        L.kv8_attention(s["q"], s["handle"], s["table"], s["seq"], c["bs"], c["K"], c["draft"], 0, c["nq"],
                        s["split"][0], s["split"][1], s["out"], s["ws"], status=s["status"])
        return [s["out"]]
    L.token_logprobs(s["logits"], s["ids"], s["logprob"], s["entropy"], s["rank"], top_logprob=s["top"],
                     top_ids=s["top_ids"], temperature=s["temperature"], status=s["status"])
    return [s["logprob"], s["entropy"], s["rank"], s["top"], s["top_ids"]]


# ---------------------------------------------------------------------- work
def work(case):
    kind = case["kind"]
    if kind in ("store", "load"):
        n, nkv = case["m"] if kind == "store" else case["n"], case["nkv"]
        held = 2 * nkv * (2 * D if case["fmt"] == "bf16" else D + 1)   # one token's K and V as the cache holds them
        if kind == "load":
            return {"bytes": n * (held + 4 * nkv * D + 8), "flops": 2 * n * nkv * D}
        nq = case["nq"]
        pos = 12 if case["mrope"] else 4
        # rows and positions in; q, the cache's rows and the values read back out
        return {"bytes": n * ((nq + 2 * nkv) * D * 2 + pos + 8 + nq * D * 2 + held + 4 * nkv * D),
                "flops": n * (nq + nkv) * (4 * D * case["norm"] + 3 * case["rd"]) + 4 * n * nkv * D}
    if kind == "attend":
        nq, nkv, K = case["nq"], case["nkv"], case["K"]
        lens = _lens(case)
        seen = sum(sum(_limits(case, n - K)) for n in lens)
        return {"bytes": sum(lens) * 2 * nkv * (D + 1) + sum((n + PAGE - 1) // PAGE * 4 + 8 for n in lens)
                + 2 * len(lens) * K * nq * D * 2, "flops": 4 * seen * nq * D}
    rows, vocab = case["rows"], case["vocab"]
    size = 2 if case["dtype"] == "bf16" else 4
    return {"bytes": rows * (vocab * size + 8 + 12 + 8 * case["n_top"] + 4 * case["warm"]), "flops": 5 * rows * vocab}


# ---------------------------------------------------------------------- the definitions in 64 bits
def _grid(fmt):
    """Every non-negative value a code can take, ascending (index parity = parity of the code)."""
    if fmt == "int8":
        return torch.arange(128, dtype=torch.float64, device="cuda")
    v = [m / 512 for m in range(8)] + [(8 + m) / 8 * 2.0 ** (k - 7) for k in range(1, 16) for m in range(8)]
    return torch.tensor(v[:127], dtype=torch.float64, device="cuda")


def _nearest(y, grid):
    """|y| to the nearest grid value, ties to the even code."""
    a = y.abs().contiguous()
    hi = torch.searchsorted(grid, a).clamp_max(grid.numel() - 1)
    lo = (hi - 1).clamp_min(0)
    dh, dl = grid[hi] - a, a - grid[lo]
    pick = torch.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    return torch.sign(y) * grid[torch.where(a >= grid[-1], torch.full_like(pick, grid.numel() - 1), pick)]


def _two64(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _held64(y, fmt):
    """What the cache holds for rows y [..., 128] (float64)."""
    top = {"e4m3": 448.0, "int8": 127.0}[fmt]
    borders = top * _two64(torch.arange(E_MIN, E_MAX, device="cuda"))
    scale = _two64(E_MIN + torch.searchsorted(borders, y.abs().amax(-1).contiguous()))[..., None]
    return _nearest(y / scale, _grid(fmt)) * scale


def _exact_store(s):
    c = s["case"]
    m, nq, nkv, rd = c["m"], c["nq"], c["nkv"], c["rd"]
    x = s["qkv"].double().view(m, -1, D)
    f = s["inv_freq"].double()
    ang = torch.empty((m, rd // 2), dtype=torch.float64, device="cuda")
    if c["mrope"]:
        i = 0
        for ax, n in enumerate(s["section"]):
            ang[:, i: i + n] = s["row_pos3"][:, ax: ax + 1].double() * f[i: i + n]
            i += n
    else:
        ang[:] = torch.outer(s["row_pos"].double(), f)
    turn = torch.polar(torch.ones_like(ang), ang)[:, None]

    def rotated(y, w):
        if w is not None:
            y = y / torch.sqrt(torch.linalg.vecdot(y, y)[..., None] / D + EPS) * w.double()
        r = y[..., :rd]
        pair = r.unflatten(-1, (2, rd // 2)).transpose(-1, -2) if c["half"] else r.unflatten(-1, (rd // 2, 2))
        z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
        z = z.transpose(-1, -2).flatten(-2) if c["half"] else z.flatten(-2)
        return torch.cat([z, y[..., rd:]], -1)

    q = rotated(x[:, :nq], s["q_norm"])
    k = rotated(x[:, nq: nq + nkv], s["k_norm"])
    v = x[:, nq + nkv:]
    if c["fmt"] != "bf16":
        k, v = _held64(k, c["fmt"]), _held64(v, c["fmt"])
    return [q.reshape(m, -1), k.reshape(m, -1), v.reshape(m, -1)]


def _rows64(codes, exps, slot):
    """Cache rows by slot in 64 bits: [n, heads, 128]."""
    flat = codes.double().transpose(1, 2).flatten(0, 1)[slot]
    return flat if exps is None else flat * _two64(exps).transpose(1, 2).flatten(0, 1)[slot][..., None]


def _exact_attend(s):
    c = s["case"]
    K, nq, nkv = c["K"], c["nq"], c["nkv"]
    G = nq // nkv
    ck, cv, ke, ve = s["cache"]
    rows = []
    for b, n in enumerate(s["lens"]):
        pages = s["table"][b, : (n + PAGE - 1) // PAGE].long()
        local = torch.arange(n, device="cuda")
        k = _rows64(ck[pages], ke[pages], local)
        v = _rows64(cv[pages], ve[pages], local)
        q = s["q"][b * K: (b + 1) * K].double().view(K, nkv, G, D)
        for j, lim in enumerate(_limits(c, n - K)):
            sc = torch.einsum("hgd,thd->hgt", q[j], k[:lim]) / D ** 0.5
            rows.append(torch.einsum("hgt,thd->hgd", torch.softmax(sc, -1), v[:lim]).reshape(nq * D))
    return [torch.stack(rows)]


def _exact_logprobs(s):
    c = s["case"]
    outs = []
    for r in range(0, c["rows"], 64):
        raw = s["logits"][r: r + 64].double()
        ids = s["ids"][r: r + 64]
        x = raw if s["temperature"] is None else raw / s["temperature"][r: r + 64, None].double()
        lp = torch.log_softmax(x, 1)
        p = lp.exp()
        ent = -(p * torch.where(p > 0, lp, torch.zeros_like(lp))).sum(1)
        order = torch.sort(raw, dim=1, descending=True, stable=True).indices
        rank = (order == ids[:, None]).long().argmax(1) + 1
        top_ids = order[:, : c["n_top"]]
        outs.append((lp.gather(1, ids[:, None])[:, 0], ent, rank.to(torch.int32), lp.gather(1, top_ids),
                     top_ids.to(torch.int32)))
    return [torch.cat(t) for t in zip(*outs)]


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "store":
        return _exact_store(s)
    if case["kind"] == "load":
        return [_rows64(c, e, s["slot"]).reshape(case["n"], -1) for c, e in (s["cache"][0::2], s["cache"][1::2])]
    return _exact_attend(s) if case["kind"] == "attend" else _exact_logprobs(s)
