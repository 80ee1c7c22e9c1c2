"""8-bit K/V cache on a B200: the write, the read-back and the attention against the 64-bit oracle.  Cached codes and
exponents have to equal the oracle's; computed outputs stay within bounds derived from the arithmetic beside each test."""
import math

import pytest
import torch

from gravityocr_b200 import _lib as L
from oracle import kv8_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
DT = {"bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "int8": torch.int8}
BF16 = 2.0 ** -8   # half a step, relative
HALF = 2.0 ** -11


def _cache(pages, nkv, fmt, fill=0):
    """Tensors of a cache whose every byte is `fill`."""
    n = 2 if fmt == "bf16" else 1
    k, v = (torch.full((pages, nkv, 16, 128 * n), fill, dtype=torch.uint8, device=DEV).view(DT[fmt]) for _ in range(2))
    if fmt == "bf16":
        return k, v, None, None
    ke, ve = (torch.full((pages, nkv, 16), fill, dtype=torch.uint8, device=DEV).view(torch.int8) for _ in range(2))
    return k, v, ke, ve


def _rows(t, slots):
    """Cache rows by slot on the CPU: [n, heads, ...]."""
    t = t.cpu()
    if t.dtype == torch.float8_e4m3fn:
        t = t.to(torch.float32)
    return t.transpose(1, 2).flatten(0, 1)[slots.cpu()]


def _status():
    return torch.zeros((1,), dtype=torch.int32, device=DEV)


def _write_case(m, fmt, half, rd, norm, mrope, nq, nkv, far=4096, extra=0, seed=0):
    g = torch.Generator().manual_seed(seed + m)
    width = (nq + 2 * nkv) * 128
    x = torch.randn((m, width + extra), generator=g) * torch.exp(torch.randn((m, 1), generator=g))
    pages = m // 16 + 3
    return dict(
        qkv=x.bfloat16().to(DEV)[:, :width], fmt=fmt, half=half, rd=rd, nq=nq, nkv=nkv, m=m, pages=pages,
        inv=(1.0 / 10000.0 ** (torch.arange(0, rd, 2, dtype=torch.float64) / max(rd, 1))).float(),
        pos=None if mrope or not rd else torch.randint(0, far, (m,), generator=g, dtype=torch.int32),
        pos3=torch.randint(0, far, (m, 3), generator=g, dtype=torch.int32) if mrope else None,
        section=(rd // 8, rd // 4, rd // 2 - rd // 8 - rd // 4) if mrope else None,
        qn=(1 + 0.2 * torch.randn(128, generator=g)).bfloat16() if norm else None,
        kn=(1 + 0.2 * torch.randn(128, generator=g)).bfloat16() if norm else None,
        slots=torch.randperm(pages * 16, generator=g)[:m])


def _write(c, cache, status=None, slots=None, q=None, stream=None):
    up = lambda t: None if t is None else t.to(DEV)
    if q is None:
        q = torch.full((c["m"], c["nq"] * 128), float("nan"), dtype=torch.bfloat16, device=DEV)
    L.qk_norm_rope_write(c["qkv"], c["nq"], L.kv_cache(*cache), up(c["slots"] if slots is None else slots), q, up(c["inv"]),
                         c["rd"], row_pos=up(c["pos"]), row_pos3=up(c["pos3"]), mrope_section=c["section"],
                         rope_half=c["half"], q_norm=up(c["qn"]), k_norm=up(c["kn"]), eps=1e-6, status=status,
                         stream=stream)
    return q


def _write_ref(c):
    m, nq, nkv = c["m"], c["nq"], c["nkv"]
    x = c["qkv"].cpu().double().view(m, nq + 2 * nkv, 128)
    ang = R.angles(c["inv"], c["pos"], c["pos3"], c["section"]) if c["rd"] else None
    return (R.norm_rotate(x[:, :nq], c["qn"], 1e-6, ang, c["half"]),
            R.norm_rotate(x[:, nq: nq + nkv], c["kn"], 1e-6, ang, c["half"]), x[:, nq + nkv:])


def _close_bf16(got, ref):
    # one rounding to bf16; before it fp32: a 128-term sum, rsqrt and four products, below 32 * 2^-24 of the row's largest
    tol = BF16 * ref.abs() + 2.0 ** -19 * ref.abs().amax(-1, keepdim=True)
    assert ((got.double().cpu().view(ref.shape) - ref).abs() <= tol).all()


WRITES = [
    (1, "int8", False, 64, True, False, 16, 8), (1, "e4m3", True, 128, False, False, 16, 8),
    (3, "bf16", False, 32, True, True, 4, 4), (17, "e4m3", False, 64, False, True, 16, 8),
    (130, "int8", True, 96, True, False, 5, 1), (257, "int8", False, 0, True, False, 2, 2),
    (257, "e4m3", True, 16, True, True, 7, 7), (33, "int8", False, 8, True, True, 3, 1), (1000, "bf16", True, 128, False, False, 16, 2),
    (2500, "int8", False, 128, True, True, 12, 4), (2500, "e4m3", False, 64, True, False, 16, 8),
    (4401, "int8", True, 64, True, False, 3, 1),   # more rows than run at once
]


@pytest.mark.parametrize("m,fmt,half,rd,norm,mrope,nq,nkv", WRITES)
def test_write(m, fmt, half, rd, norm, mrope, nq, nkv):
    c = _write_case(m, fmt, half, rd, norm, mrope, nq, nkv, far=300000, extra=128 if m % 2 else 0)
    cache = _cache(c["pages"], nkv, fmt, fill=0x55)
    st = _status()
    q = _write(c, cache, st)
    torch.cuda.synchronize()
    assert int(st) == 0
    rq, rk, rv = _write_ref(c)
    _close_bf16(q, rq)
    k, v, ke, ve = cache
    if fmt == "bf16":
        _close_bf16(_rows(k, c["slots"]), rk)
        assert torch.equal(_rows(v, c["slots"]).double(), rv)
    else:
        for ref, codes, exps in ((rk, k, ke), (rv, v, ve)):
            want, e = R.quantise(ref, fmt)
            assert torch.equal(_rows(exps, c["slots"]).long(), e)
            assert torch.equal(_rows(codes, c["slots"]).double(), want)
    # slots that no row names keep every byte
    free = torch.tensor(sorted(set(range(c["pages"] * 16)) - set(c["slots"].tolist())))
    for t in cache:
        if t is not None:
            assert (_rows(t.view(torch.uint8), free) == 0x55).all()


@pytest.mark.parametrize("fmt", ["bf16", "e4m3", "int8"])
def test_write_skips_rows_without_a_slot(fmt):
    c = _write_case(9, fmt, False, 64, False, False, 4, 2)
    cache = _cache(c["pages"], 2, fmt, fill=0x11)
    slots = c["slots"].clone()
    slots[[0, 4, 8]] = -1
    st = _status()
    q = _write(c, cache, st, slots=slots)
    assert int(st) == 0
    _close_bf16(q, _write_ref(c)[0])     # q is written for every row
    for s in c["slots"][[0, 4, 8]].tolist():
        assert (cache[0].view(torch.uint8)[s // 16, :, s % 16] == 0x11).all()
    slots[2] = c["pages"] * 16           # past the cache: refused on the device, the rest of the rows go on
    _write(c, cache, st, slots=slots)
    assert int(st) == 6
    if fmt != "bf16":
        assert torch.equal(_rows(cache[3], slots[[1, 3]]).long(), R.quantise(_write_ref(c)[2], fmt)[1][[1, 3]])


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_write_special_rows(fmt):
    """Zeros, NaN, infinities, a lone loud element, values past the exponents' range, borders and ties."""
    nkv = 1
    rows = torch.zeros((12, 3, 128))
    rows[1, 1:, 5] = float("nan")
    rows[2, 1:, 100] = float("inf")
    rows[3, 1:, 0] = float("-inf")
    rows[4, 1:] = 1e-3
    rows[4, 1:, 77] = 1000.0
    rows[5, 1:] = 2.0 ** 60
    rows[6, 1:] = 2.0 ** -60
    rows[7, 1:] = R.TOP[fmt]
    rows[8, 1:] = R.TOP[fmt] + 1.0
    rows[9, 1:] = torch.arange(128) * 0.5 - 32          # ties of the int8 grid
    rows[9, 1:, 0] = R.TOP[fmt]
    g = R.grid("e4m3")
    rows[10, 1:, :126] = ((g[1:] + g[:-1]) / 2).float()  # ties of the e4m3 grid
    rows[11, 1:] = -rows[10, 1:]
    c = _write_case(12, fmt, False, 0, False, False, 1, nkv)
    c["qkv"] = rows.bfloat16().view(12, 384).to(DEV)
    cache = _cache(c["pages"], nkv, fmt, fill=0x33)
    _write(c, cache)
    _, rk, rv = _write_ref(c)
    for ref, codes, exps in ((rk, cache[0], cache[2]), (rv, cache[1], cache[3])):
        want, e = R.quantise(ref, fmt)
        assert torch.equal(_rows(exps, c["slots"]).long(), e)
        assert torch.equal(_rows(codes, c["slots"]).double(), want)
    out = torch.zeros((2, 12, 128), dtype=torch.bfloat16, device=DEV)
    L.kv_read(L.kv_cache(*cache), c["slots"].to(DEV), out[0], out[1])
    for o in out.cpu():
        assert torch.isnan(o[1:4].float()).all() and torch.isfinite(o[[0, *range(4, 12)]].float()).all()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_write_k_maxima_next_to_the_exponents_border(fmt, half):
    """Rotated k rows whose largest value is top 2^j (1 + d): d = 0, and within 10^-5 .. 10^-14 above and below, of both signs."""
    d = [0.0] + [s * 10.0 ** -n for n in range(5, 15) for s in (1, -1)]
    m = 2 * len(d)
    c = _write_case(m, fmt, half, 128, False, False, 2, 2)
    rows = torch.randn((m, 6, 128), generator=torch.Generator().manual_seed(5))
    i, j = (0, 64) if half else (0, 1)
    rows[:, :, i] = R.TOP[fmt] * (2.0 ** (torch.arange(m) % 7 - 3))[:, None]
    rows[1::2, :, i] *= -1
    rows[:, :, j] = -rows[:, :, i] / 128                # d moves it by the angle's 128th
    c["qkv"] = rows.bfloat16().view(m, 768).to(DEV)
    for k, x in enumerate(d):                            # y_i = x_i cos - x_j sin = x_i (1 + a / 128 - ..): a = 128 d
        inv = torch.zeros(64)
        inv[0] = 128 * x
        c["inv"] = inv
        c["pos"] = torch.ones(m, dtype=torch.int32)
        cache = _cache(c["pages"], 2, fmt)
        _write(c, cache)
        want, e = R.quantise(_write_ref(c)[1], fmt)
        assert torch.equal(_rows(cache[2], c["slots"]).long(), e), x
        assert torch.equal(_rows(cache[0], c["slots"]).double(), want), x


def test_write_row_does_not_depend_on_its_batch():
    c = _write_case(2500, "e4m3", True, 64, True, False, 16, 8)
    a, b = _cache(c["pages"], 8, "e4m3"), _cache(c["pages"], 8, "e4m3")
    qa = _write(c, a)
    qb = torch.zeros_like(qa)
    for lo, hi in ((0, 1), (1, 40), (40, 2500)):
        part = dict(c, qkv=c["qkv"][lo:hi], m=hi - lo, slots=c["slots"][lo:hi], pos=c["pos"][lo:hi])
        _write(part, b, q=qb[lo:hi])
    assert torch.equal(qa, qb)
    for x, y in zip(a, b):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


@pytest.mark.parametrize("n,fmt,nkv", [(1, "e4m3", 8), (7, "int8", 1), (301, "bf16", 3), (333, "e4m3", 5),
                                       (5000, "int8", 8), (5000, "bf16", 2)])
def test_read(n, fmt, nkv):
    g = torch.Generator().manual_seed(n)
    pages = n // 16 + 5
    raw = torch.randint(0, 256, (2, pages, nkv, 16, 128 * (2 if fmt == "bf16" else 1)), generator=g, dtype=torch.uint8)
    if fmt == "e4m3":
        raw[(raw & 0x7F) == 0x7F] = 0x7E    # no NaN codes: the write makes none
    k, v = (t.to(DEV).view(DT[fmt]) for t in raw)
    ke = ve = None
    if fmt != "bf16":
        ke, ve = (torch.randint(-40, 41, (pages, nkv, 16), generator=g).to(DEV, torch.int8) for _ in range(2))
        ke[1, 0, 3] = -128
    slots = torch.randint(0, pages * 16, (n,), generator=g)   # repeats are fine
    slots[n // 2] = -1 if n > 1 else slots[0]
    out = torch.full((2, n, nkv * 128), 7.0, dtype=torch.bfloat16, device=DEV)
    st = _status()
    L.kv_read(L.kv_cache(k, v, ke, ve), slots.to(DEV), out[0], out[1], status=st)
    assert int(st) == 0
    keep = slots >= 0
    for o, codes, e in ((out[0], k, ke), (out[1], v, ve)):
        o = o.cpu().view(n, nkv, 128)
        if fmt == "bf16":
            assert torch.equal(o[keep].view(torch.int16), _rows(codes, slots[keep]).view(torch.int16))
        else:
            want = R.values(_rows(codes, slots[keep]), _rows(e, slots[keep]))
            torch.testing.assert_close(o[keep].double(), want, rtol=0, atol=0, equal_nan=True)
        assert (o[~keep] == 7.0).all()
    slots[0] = pages * 16
    L.kv_read(L.kv_cache(k, v, ke, ve), slots.to(DEV), out[0], out[1], status=st)
    assert int(st) == 6


# ---------------------------------------------------------------------- attention
def _fill(fmt, pages, nkv, g, spread=1.0):
    """Quantised random rows in every slot: tensors on the GPU and their float64 values [pages * 16, heads, 128]."""
    out, vals = [], []
    for _ in range(2):
        x = torch.randn((pages, nkv, 16, 128), generator=g, dtype=torch.float64)
        x = (x * torch.exp(spread * torch.randn((pages, nkv, 16, 1), generator=g, dtype=torch.float64))).bfloat16().double()
        codes, e = R.quantise(x, fmt)
        out.append((codes.float().to(DT[fmt]).to(DEV), e.to(torch.int8).to(DEV)))
        vals.append(R.values(codes, e).transpose(1, 2).flatten(0, 1))
    (k, ke), (v, ve) = out
    return (k, v, ke, ve), vals


def _attn_case(fmt, lens, K, nq, nkv, spread=1.0, seed=0, q_scale=1.0):
    """lens: committed tokens of each request (the K window rows follow)."""
    g = torch.Generator().manual_seed(seed + 13 * len(lens) + K)
    bs = len(lens)
    need = [max(1, -(-(n + K) // 16)) for n in lens]
    pages = sum(need) + 3
    cache, (kv, vv) = _fill(fmt, pages, nkv, g, spread)
    perm = torch.randperm(pages, generator=g).to(torch.int32)
    pt = torch.full((bs, max(need) + 1), 2 ** 30, dtype=torch.int32)   # entries past a request's pages are never read
    slots, o = [], 0
    for b in range(bs):
        pt[b, : need[b]] = perm[o: o + need[b]]
        o += need[b]
        t = torch.arange(max(0, lens[b] + K))
        slots.append(pt[b].long()[t // 16] * 16 + t % 16)
    q = (torch.randn((bs * K, nq * 128), generator=g) * q_scale).bfloat16()
    return dict(cache=cache, k=kv, v=vv, pt=pt.to(DEV), slots=slots, q=q, lens=list(lens), K=K, nq=nq, nkv=nkv, bs=bs)


def _attend(c, draft=0, base_add=0, chunk=None, splits=None, status=None, ws=None, out=None, stream=None):
    longest = max(1, max(c["lens"]) + c["K"])
    if chunk is None:
        chunk, splits = L.kv8_attention_split(c["bs"], c["K"], longest, c["nq"], c["nkv"])
    elif splits is None:
        splits = -(-longest // chunk)
    if ws is None:
        ws = torch.zeros((L.kv8_attention_workspace_bytes(c["bs"], c["K"], c["nq"], c["nkv"], splits),),
                         dtype=torch.uint8, device=DEV)
    if out is None:
        out = torch.full((c["bs"] * c["K"], c["nq"] * 128), float("nan"), dtype=torch.bfloat16, device=DEV)
    L.kv8_attention(c["q"].to(DEV), L.kv_cache(*c["cache"]), c["pt"],
                    torch.tensor(c["lens"], dtype=torch.int64, device=DEV) - base_add, c["bs"], c["K"], draft, base_add,
                    c["nq"], chunk, splits, out, ws, status=status, stream=stream)
    return out


def _check_attention(c, out, draft=0):
    K, nq, nkv = c["K"], c["nq"], c["nkv"]
    got = out.double().cpu().view(c["bs"], K, nq, 128)
    for b in range(c["bs"]):
        q = c["q"][b * K: (b + 1) * K].double().view(K, nq, 128)
        k, v = c["k"][c["slots"][b]], c["v"][c["slots"][b]]
        ref = R.attention(q, k, v, c["lens"][b], draft)
        if k.shape[0] == 0:
            assert (got[b] == 0).all()
            continue
        # |out - ref| <= half a bf16 step, and of sum p |v|: the rounding of p to three e4m3 parts (2^-12), fp32 sums over the
        # tokens (16 at a time, and a few joins), and twice the relative error of a weight, which is the absolute error of
        # its score: 128 products of fp32 accumulation (twice, for truncating accumulators), the exponent's argument, and q's
        # parts: 2^-21 of its largest element for e4m3, 0.5 / 32639 of it for int8's two digits
        n, G = k.shape[0], nq // nkv
        av = R.attention(q, k, v.abs(), c["lens"][b], draft)
        ka = k.abs().repeat_interleave(G, 1)
        mag = torch.einsum("jhd,thd->jht", q.abs(), ka).amax(-1, keepdim=True) / math.sqrt(128)
        int8 = c["cache"][0].dtype == torch.int8
        parts = (0.5 / 32639 if int8 else 2.0 ** -21) * q.abs().amax(-1, keepdim=True) * ka.sum(-1).amax(0)[None, :, None] / math.sqrt(128)
        arg = 1.45 * mag + 100.0
        rel = HALF + (n / 16 + 40) * 2.0 ** -23 + 2 * (256 * 2.0 ** -24 * mag + parts + 2.0 ** -22 + 4 * 2.0 ** -24 * arg)
        err = (got[b] - ref).abs()
        # a weight's absolute floor is relative to the largest weight w 2^ev of its tile, times a code <= top, and
        # top 2^ev < 2 max|v| of the largest one's row: 2^-26 for three e4m3 parts (any signs); int8's two digits round to
        # 2^-16 of it independently, so their sum over n tokens stays within 6 / sqrt(3) * 2^-15 * sqrt(n)
        loud = R.attention(q, k, v.abs().amax(-1, keepdim=True).expand(v.shape), c["lens"][b], draft)
        floor = 2.0 ** -13 * math.sqrt(n) if int8 else 2.0 ** -25 * n
        tol = BF16 * ref.abs() + rel * av + floor * loud
        assert (err <= tol).all(), (b, float((err / tol.clamp_min(1e-30)).max()))


ATTN = [
    # fmt, committed lengths, K, q heads, kv heads
    ("e4m3", [0], 1, 16, 8), ("int8", [0, 1, 2, 14, 15, 16, 17, 30, 31, 32, 33], 1, 16, 8),
    ("int8", [2738], 1, 16, 8), ("e4m3", [127, 128, 129, 500, 1023], 1, 5, 1), ("e4m3", [700, 3, 64], 1, 32, 2),
    ("int8", [300], 1, 128, 1), ("int8", [0, 5, 95], 2, 16, 8), ("e4m3", [63, 64, 200], 17, 16, 8),
    ("int8", [1, 400], 17, 16, 8), ("e4m3", [250], 33, 6, 3), ("int8", [31, 250], 9, 12, 4), ("e4m3", [77], 64, 4, 2),
    ("int8", [150], 128, 2, 2), ("int8", [40] * 70, 1, 4, 4),
]


@pytest.mark.parametrize("fmt,lens,K,nq,nkv", ATTN)
@pytest.mark.parametrize("draft", [0, 1, 2])
def test_attention(fmt, lens, K, nq, nkv, draft):
    c = _attn_case(fmt, lens, K, nq, nkv)
    st = _status()
    out = _attend(c, draft, status=st)
    assert int(st) == 0
    _check_attention(c, out, draft)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("K,chunk,splits", [(1, 32, None), (1, 32, 128), (1, 64, None), (1, 96, None), (1, 160, 40),
                                            (1, 1024, None), (1, 1056, 1), (17, 32, None), (17, 256, None), (5, 512, 4)])
def test_attention_splits(fmt, K, chunk, splits):
    """The same rows through every cut, the workspace used again: its tickets come back to zero."""
    c = _attn_case(fmt, [999, 0, 31, 512, 4], K, 16, 8)
    n = splits or -(-(999 + K) // chunk)
    ws = torch.full((L.kv8_attention_workspace_bytes(5, K, 16, 8, n),), 0xFF, dtype=torch.uint8, device=DEV)
    ws[:65536] = 0
    st = _status()
    first = _attend(c, chunk=chunk, splits=n, ws=ws, status=st)
    _check_attention(c, first)
    for _ in range(5):
        assert torch.equal(first, _attend(c, chunk=chunk, splits=n, ws=ws, status=st))
    assert int(st) == 0
    assert int(ws[:65536].sum()) == 0


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("K,nkv,group", [(1, 8, 2), (1, 8, 1), (3, 8, 2), (4, 8, 2), (1, 8, 5), (6, 8, 2), (3, 8, 3), (8, 8, 2),
                                         (9, 8, 2), (12, 8, 2), (25, 8, 1), (17, 8, 2), (7, 8, 5), (20, 8, 2), (41, 8, 1)])
def test_attention_row_counts(fmt, K, nkv, group):
    """Every split of the rows between thread groups, for more CTAs than run at once and for few."""
    lens = [(37 * b) % 150 for b in range(76)]
    c = _attn_case(fmt, lens, K, group * nkv, nkv)
    out = _attend(c)
    cut = dict(c, pt=c["pt"][:9].contiguous(), q=c["q"][: 9 * K], lens=lens[:9], bs=9)
    few = _attend(cut)
    _check_attention(cut, few)
    _check_attention(cut, out[: 9 * K])
    c["slots"], c["lens"] = c["slots"][-9:], c["lens"][-9:]
    _check_attention(dict(c, q=c["q"][-9 * K:], bs=9), out[-9 * K:])


@pytest.mark.parametrize("bs", [20, 255, 256, 257])
@pytest.mark.parametrize("fmt,K", [("int8", 17), ("e4m3", 20)])
def test_attention_of_many_requests_is_each_ones_own(fmt, K, bs):
    """Whatever order the requests run in (mixed, equal, empty and padding ones, more or fewer than are sorted), each gets the
    rows that it gets alone, and the tickets come back to zero."""
    g = torch.Generator().manual_seed(bs)
    lens = torch.randint(0, 700, (bs,), generator=g).tolist()
    lens[1], lens[2], lens[3], lens[bs - 1] = 0, -K, lens[5], 699
    c = _attn_case(fmt, lens, K, 16, 8)
    ws = torch.zeros((L.kv8_attention_workspace_bytes(bs, K, 16, 8, 3),), dtype=torch.uint8, device=DEV)
    st = _status()
    out = _attend(c, chunk=256, splits=3, ws=ws, status=st)
    assert int(st) == 0 and int(ws[:65536].sum()) == 0
    for b in sorted({0, 1, 2, 3, 5, bs - 1, *torch.randint(0, bs, (12,), generator=g).tolist()}):
        one = dict(c, pt=c["pt"][b: b + 1].contiguous(), q=c["q"][b * K: (b + 1) * K], lens=[lens[b]], bs=1)
        assert torch.equal(out[b * K: (b + 1) * K], _attend(one, chunk=256, splits=3)), b
    if bs == 20:
        _check_attention(c, out)
        # beyond a short plan, and beyond the page table: reported, the other requests as before
        for cut, code in ((2, 1), (3, 6)):
            short = dict(c, pt=c["pt"] if cut == 2 else c["pt"][:, :30].contiguous())
            st.zero_()
            got = _attend(short, chunk=256, splits=cut, ws=ws, status=st)
            assert int(st) == code and int(ws[:65536].sum()) == 0
            for b in range(bs):
                if lens[b] + K <= 480:
                    assert torch.equal(got[b * K: (b + 1) * K], out[b * K: (b + 1) * K])


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_attention_peaked_and_flat_scores(fmt):
    for q_scale in (0.0, 8.0):
        c = _attn_case(fmt, [1500, 40], 1, 16, 8, q_scale=q_scale)
        _check_attention(c, _attend(c))


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("chunk", [8192, 1024])
def test_attention_one_loud_token_and_many_quiet_ones(fmt, chunk):
    """The first token takes half of the attention, 20,000 others the rest between them, and their values share a mean: no
    token's weight may vanish next to the first one's."""
    n = 20000
    c = _attn_case(fmt, [n - 1], 1, 2, 1, spread=0.0)
    k, v, ke, ve = c["cache"]
    pages = k.shape[0]
    g = torch.Generator().manual_seed(1)
    q = c["q"].double().view(2, 128)
    xk = 0.05 * torch.randn((pages * 16, 128), generator=g, dtype=torch.float64)
    dirn = torch.linalg.pinv(q) @ torch.full((2, 1), math.log(n) * math.sqrt(128), dtype=torch.float64)
    xk[int(c["slots"][0][0])] = dirn[:, 0]
    xv = (1.0 + 0.3 * torch.randn((pages * 16, 128), generator=g, dtype=torch.float64))
    for x, codes, exps, name in ((xk, k, ke, "k"), (xv, v, ve, "v")):
        qc, e = R.quantise(x.view(pages, 1, 16, 128), fmt)
        codes.copy_(qc.float().to(DT[fmt]))
        exps.copy_(e.to(torch.int8))
        c[name] = R.values(qc, e).transpose(1, 2).flatten(0, 1)
    _check_attention(c, _attend(c, chunk=chunk))


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_attention_exponents_far_apart(fmt):
    """Values whose exponents span the format's range: the softmax sum must not lose the quiet rows."""
    c = _attn_case(fmt, [200], 1, 4, 2, spread=0.0)
    k, v, ke, ve = c["cache"]
    e = torch.randint(-40, 41, ve.shape, generator=torch.Generator().manual_seed(3)).to(torch.int8)
    ve.copy_(e)
    codes = v.cpu().to(torch.float32).double()
    c["v"] = R.values(codes, e).transpose(1, 2).flatten(0, 1)
    _check_attention(c, _attend(c))
    # only the quietest rows
    ve.fill_(-40)
    c["v"] = R.values(codes, ve.cpu()).transpose(1, 2).flatten(0, 1)
    _check_attention(c, _attend(c))


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_attention_ignores_what_it_does_not_see(fmt):
    """Slots past a request's rows hold NaN codes and bad exponents; window rows hidden by the causal mask are bad rows."""
    c = _attn_case(fmt, [5, 33, 100, 0], 3, 16, 8)
    seen = torch.cat(c["slots"])
    hidden = torch.ones(c["k"].shape[0], dtype=torch.bool)
    hidden[seen] = False
    hidden = hidden.view(-1, 16).to(DEV)
    for t in c["cache"][:2]:
        t.view(torch.uint8).transpose(1, 2)[hidden] = 0xFF
    for t in c["cache"][2:]:
        t.transpose(1, 2)[hidden] = -128
    _check_attention(c, _attend(c))
    # the last window row of request 1 is a bad row: rows 0 and 1 do not see it, row 2 does
    s = int(c["slots"][1][-1])
    c["cache"][3][s // 16, :, s % 16] = -128
    out = _attend(c).view(4, 3, -1)
    assert torch.isfinite(out[1, :2].float()).all() and torch.isnan(out[1, 2].float()).all()
    assert torch.isfinite(out[[0, 2, 3]].float()).all()
    c["cache"][3][s // 16, :, s % 16] = 0
    c["cache"][2][s // 16, 3, s % 16] = -128          # a bad key of one head
    out = _attend(c).view(4, 3, 8, 2, 128)
    assert torch.isnan(out[1, 2, 3].float()).all()
    assert torch.isfinite(out[1, 2, [0, 1, 2, 4, 5, 6, 7]].float()).all() and torch.isfinite(out[1, :2].float()).all()


def test_attention_rows_that_see_nothing():
    """Padding requests (length -K) and rows before the first token give zeros, also next to real ones."""
    c = _attn_case("int8", [-2, 40, -1], 2, 16, 8)
    out = _attend(c)
    _check_attention(dict(c, bs=1, lens=[40], slots=[c["slots"][1]], q=c["q"][2:4]), out[2:4])
    assert (out[:2] == 0).all() and (out[4] == 0).all()
    # request 2's second row sees its own token: the weights are one, the output is that token's values
    want = c["v"][c["slots"][2]].repeat_interleave(2, 1).view(-1)
    assert ((out[5].double().cpu() - want).abs() <= BF16 * want.abs() + 2.0 ** -20 * want.abs()).all()
    assert (_attend(_attn_case("e4m3", [-1], 1, 16, 8), chunk=32) == 0).all()


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("K", [1, 17])
def test_attention_huge_scores(fmt, K):
    """Scores of tens of thousands (base 2), where a score's fp32 step is a good part of a percent of a weight: the largest
    weight of a tile must not wrap, and each row still attends to its largest scores alone."""
    c = _attn_case(fmt, [700, 130], K, 16, 8, spread=0.0)
    c["q"] = (c["q"].float() * 4000).bfloat16()
    out = _attend(c).double().cpu().view(2, K, 16, 128)
    for b in range(2):
        q = c["q"][b * K: (b + 1) * K].double().view(K, 16, 128)
        k, v = c["k"][c["slots"][b]], c["v"][c["slots"][b]]
        s = torch.einsum("jhd,thd->jht", q, k.repeat_interleave(2, 1)) / math.sqrt(128) * 1.4427
        lim = torch.tensor(R.row_limits(0, c["lens"][b], K))
        s[(torch.arange(k.shape[0])[None] >= lim[:, None])[:, None].expand(s.shape)] = -math.inf
        top = torch.topk(s, 2, -1)
        sure = top.values[..., 0] - top.values[..., 1] > 64    # all the weight on one token, whatever the rounding
        assert sure.float().mean() > 0.5  # of the inputs, not of the kernel: most rows have a clear winner
        want = v.repeat_interleave(2, 1).transpose(0, 1)[torch.arange(16)[None], top.indices[..., 0]]
        err = (out[b] - want).abs()[sure]
        assert (err <= BF16 * want.abs()[sure] + 2.0 ** -14 * want.abs().amax(-1, keepdim=True).expand(want.shape)[sure]).all()


def test_attention_reports_a_plan_that_is_too_short():
    c = _attn_case("int8", [100, 20], 1, 16, 8)
    st = _status()
    _attend(c, chunk=64, splits=1, status=st)
    assert int(st) == 1
    st.zero_()
    _attend(c, chunk=64, splits=2, status=st)
    assert int(st) == 0


def test_attention_reports_bad_pages():
    c = _attn_case("int8", [100, 30], 1, 16, 8)
    st = _status()
    c["pt"][0, 2] = c["cache"][0].shape[0]
    out = _attend(c, status=st)
    assert int(st) == 6
    _check_attention(dict(c, bs=1, lens=[30], slots=c["slots"][1:], q=c["q"][1:]), out[1:])
    c = _attn_case("int8", [100, 30], 1, 16, 8)
    st.zero_()
    c["pt"] = c["pt"][:, :2].contiguous()      # request 0's length runs past its table
    out = _attend(c, status=st)
    assert int(st) == 6
    _check_attention(dict(c, bs=1, lens=[30], slots=c["slots"][1:], q=c["q"][1:]), out[1:])


def test_attention_past_32_bit_offsets():
    """Pages whose code offsets lie beyond 2^31 bytes."""
    pages, nkv = 2 ** 31 // (8 * 16 * 128) + 40, 8
    k, v = (torch.zeros((pages, nkv, 16, 128), dtype=torch.int8, device=DEV) for _ in range(2))
    ke, ve = (torch.zeros((pages, nkv, 16), dtype=torch.int8, device=DEV) for _ in range(2))
    g = torch.Generator().manual_seed(5)
    small, (kv, vv) = _fill("int8", 32, nkv, g)
    for big, t in zip((k, v, ke, ve), small):
        big[-32:] = t
    lens, K, nq = [400, 90], 1, 16
    pt = torch.zeros((2, 26), dtype=torch.int32)
    pt[0, :26] = torch.arange(26) + pages - 32
    pt[1, :6] = torch.arange(26, 32) + pages - 32
    slots = [torch.arange(401), 26 * 16 + torch.arange(91)]
    q = torch.randn((2, nq * 128), generator=g).bfloat16()
    c = dict(cache=(k, v, ke, ve), k=kv, v=vv, pt=pt.to(DEV), slots=slots, q=q, lens=lens, K=K, nq=nq, nkv=nkv, bs=2)
    _check_attention(c, _attend(c))
    # written and read there too
    w = _write_case(5, "int8", False, 64, False, False, 16, 8)
    w["slots"] = torch.arange(5) + (pages - 3) * 16
    _write(w, (k, v, ke, ve))
    out = torch.zeros((2, 5, nkv * 128), dtype=torch.bfloat16, device=DEV)
    L.kv_read(L.kv_cache(k, v, ke, ve), w["slots"].to(DEV), out[0], out[1])
    want, e = R.quantise(_write_ref(w)[2], "int8")
    assert torch.equal(out[1].double().cpu().view(5, nkv, 128), R.values(want, e))


# ---------------------------------------------------------------------- the operators together
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_decode_steps_write_then_attend(fmt):
    """Ten decode steps of three requests: each step writes its token and attends over the cache, in a captured graph on a
    stream of its own; every step's output is checked, and the cache holds the oracle's rows at the end."""
    nq, nkv, bs, steps, rd = 16, 8, 3, 10, 64
    g = torch.Generator().manual_seed(2)
    pages = 16
    cache = _cache(pages, nkv, fmt, fill=0xFF)
    handle = L.kv_cache(*cache)
    pt = torch.randperm(pages, generator=g)[: bs * 4].view(bs, 4).to(torch.int32)
    lens = torch.tensor([0, 7, 29])
    inv = (1.0 / 10000.0 ** (torch.arange(0, rd, 2, dtype=torch.float64) / rd)).float()
    history = [[] for _ in range(bs)]   # per request: the (k, v) rows the cache holds, float64

    qkv = torch.zeros((bs, (nq + 2 * nkv) * 128), dtype=torch.bfloat16, device=DEV)
    pos, slot = torch.zeros(bs, dtype=torch.int32, device=DEV), torch.zeros(bs, dtype=torch.int64, device=DEV)
    seq = torch.zeros(bs, dtype=torch.int64, device=DEV)
    q = torch.zeros((bs, nq * 128), dtype=torch.bfloat16, device=DEV)
    out = torch.zeros_like(q)
    chunk, splits = L.kv8_attention_split(bs, 1, 64, nq, nkv)
    chunk, splits = 32, 2
    ws = torch.zeros((L.kv8_attention_workspace_bytes(bs, 1, nq, nkv, splits),), dtype=torch.uint8, device=DEV)
    st = _status()
    inv_d, pt_d = inv.to(DEV), pt.to(DEV)

    def step():
        L.qk_norm_rope_write(qkv, nq, handle, slot, q, inv_d, rd, row_pos=pos, status=st)
        L.kv8_attention(q, handle, pt_d, seq, bs, 1, 0, 0, nq, chunk, splits, out, ws, status=st)

    def feed(x, at):
        qkv.copy_(x.to(DEV))
        pos.copy_(at.to(torch.int32))
        seq.copy_(at)
        slot.copy_(pt.gather(1, (at // 16)[:, None])[:, 0].long() * 16 + at % 16)

    def reference(x, at):
        y = x.double().view(bs, nq + 2 * nkv, 128)
        ang = R.angles(inv, at)
        rq = R.norm_rotate(y[:, :nq], None, 0.0, ang, False)
        rk = R.norm_rotate(y[:, nq: nq + nkv], None, 0.0, ang, False)
        for b in range(bs):
            history[b].append(tuple(R.values(*R.quantise(t[b], fmt)) for t in (rk, y[:, nq + nkv:])))
        return rq

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        # the prefixes: one write per token position, requests that are done pass slot -1
        for t in range(int(lens.max())):
            x = torch.randn((bs, qkv.shape[1]), generator=g).bfloat16()
            feed(x, torch.full((bs,), t))
            slot[lens.to(DEV) <= t] = -1
            L.qk_norm_rope_write(qkv, nq, handle, slot, q, inv_d, rd, row_pos=pos, status=st)
            before = [len(h) for h in history]
            reference(x, torch.full((bs,), t))
            for b in range(bs):
                if t >= int(lens[b]):
                    history[b].pop()
                    assert len(history[b]) == before[b]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step()
        for i in range(steps):
            x = torch.randn((bs, qkv.shape[1]), generator=g).bfloat16()
            feed(x, lens + i)
            graph.replay()
            reference(x, lens + i)
            stream.synchronize()
            c = dict(K=1, nq=nq, nkv=nkv, bs=1, cache=cache)
            for b in range(bs):
                k = torch.stack([h[0] for h in history[b]])
                v = torch.stack([h[1] for h in history[b]])
                _check_attention(dict(c, q=q[b: b + 1].cpu(), k=k, v=v, slots=[torch.arange(k.shape[0])],
                                      lens=[k.shape[0] - 1]), out[b: b + 1])
    assert int(st) == 0


def test_a_dropped_handle_frees_the_cache():
    import gc
    gc.collect()
    gc.disable()
    try:
        before = torch.cuda.memory_allocated()
        L.kv_cache(*_cache(64, 8, "int8"))
        assert torch.cuda.memory_allocated() == before
    finally:
        gc.enable()


def test_calls_on_two_streams_at_once():
    """Two requests' attention with a workspace each, on two streams, many times over: the same rows as one after the other."""
    a, b = _attn_case("int8", [3000], 1, 16, 8), _attn_case("e4m3", [2500], 1, 16, 8, seed=4)
    want = [_attend(c, chunk=256) for c in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, c in enumerate((a, b)):
            with torch.cuda.stream(streams[i]):
                got[i].append(_attend(c, chunk=256))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(x, w) for x in g)


def test_wrappers_refuse():
    cache = _cache(4, 2, "int8")
    h = L.kv_cache(*cache)
    q = torch.zeros((1, 256), dtype=torch.bfloat16, device=DEV)
    slots = torch.zeros((1,), dtype=torch.int64, device=DEV)
    with pytest.raises(RuntimeError, match="need k_exp"):
        L.kv_cache(cache[0], cache[1])
    with pytest.raises(RuntimeError, match="takes neither"):
        L.kv_cache(*_cache(4, 2, "bf16")[:2], cache[2], cache[3])
    with pytest.raises(RuntimeError, match="must be"):
        L.kv_cache(cache[0], cache[1], cache[2][:3], cache[3])
    with pytest.raises(RuntimeError, match="does not hold"):
        L.qk_norm_rope_write(torch.zeros((1, 640), dtype=torch.bfloat16, device=DEV), 2, h, slots, q, None, 0)
    with pytest.raises(RuntimeError, match="row_slot"):
        L.qk_norm_rope_write(torch.zeros((1, 768), dtype=torch.bfloat16, device=DEV), 2, h, slots.int(), q, None, 0)
    with pytest.raises(RuntimeError, match="k_out holds"):
        L.kv_read(h, slots, q[:, :128].contiguous(), q)
    pt = torch.zeros((1, 4), dtype=torch.int32, device=DEV)
    with pytest.raises(RuntimeError, match="fewer than"):
        L.kv8_attention(q, h, pt, slots, 2, 1, 0, 0, 2, 32, 1, q, None)
    with pytest.raises(RuntimeError, match="at least"):
        L.kv8_attention(q, h, pt.expand(2, 4).contiguous(), slots, 2, 1, 0, 0, 2, 32, 1, q, None)
    with pytest.raises(RuntimeError, match="invalid argument"):
        L.kv8_attention(q, h, pt, slots, 1, 1, 0, 0, 2, 32, 2, q, None)
