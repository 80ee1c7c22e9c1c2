"""Host side of the 8-bit K/V cache and of the log probabilities: argument checks of the C entries and the wrappers, the
split plan, the oracle's rounding."""
import ctypes

import pytest
import torch

from gravityocr_b200 import _lib as L
from oracle import kv8_ref as R
from test_abi_layout import _c_layout

ARG, UNSUPPORTED = 1, 7
P = 4096  # a pointer that no refused call follows


def _cache(**kw):
    c = L.KvCache()
    c.format, c.n_kv_heads, c.page_size, c.n_pages = L.KV_INT8, 8, 16, 64
    c.k = c.v = c.k_exp = c.v_exp = P
    for k, v in kw.items():
        setattr(c, k, v)
    return c


BAD_CACHES = [dict(format=3), dict(format=-1), dict(n_kv_heads=0), dict(page_size=1), dict(n_pages=0), dict(k=None),
              dict(v=None), dict(k_exp=None), dict(v_exp=None), dict(k=P + 8), dict(v_exp=P + 1)]


def test_cache_handle_matches_c_layout(tmp_path):
    names = [f[0] for f in L.KvCache._fields_]
    c = _c_layout("gr_kv_cache", names, tmp_path)
    assert c["size"] == ctypes.sizeof(L.KvCache)
    for n in names:
        assert c[n] == getattr(L.KvCache, n).offset, n


def _write(cache=None, **kw):
    a = dict(qkv=P, ld=32 * 128, m=4, nq=16, qn=None, kn=None, eps=1e-5, pos=P, pos3=None, sec=None, inv=P, rd=64, half=0,
             slot=P, q=P)
    a.update(kw)
    sec = None if a["sec"] is None else (ctypes.c_int32 * 3)(*a["sec"])
    return L.load().gr_qk_norm_rope_write(a["qkv"], a["ld"], a["m"], a["nq"], ctypes.byref(cache or _cache()), a["qn"],
                                          a["kn"], a["eps"], a["pos"], a["pos3"], sec, a["inv"], a["rd"], a["half"],
                                          a["slot"], a["q"], None, None)


@pytest.mark.parametrize("kw", [dict(qkv=None), dict(qkv=P + 8), dict(ld=32 * 128 - 8), dict(ld=32 * 128 + 4), dict(m=0),
                                dict(nq=0), dict(eps=-1.0), dict(eps=float("nan")), dict(pos=None), dict(inv=None),
                                dict(rd=-8), dict(rd=136), dict(rd=60), dict(rd=56, half=1), dict(slot=None), dict(q=None), dict(q=P + 8),
                                dict(qn=P + 8), dict(kn=P + 8), dict(pos3=P), dict(pos=None, pos3=P),
                                dict(pos=None, pos3=P, sec=(8, 12, 11)), dict(pos=None, pos3=P, sec=(-1, 21, 12))])
def test_write_refuses(kw):
    assert _write(**kw) == ARG


@pytest.mark.parametrize("kw", BAD_CACHES)
def test_a_broken_cache_is_refused_everywhere(kw):
    c = _cache(**kw)
    lib = L.load()
    assert _write(cache=c) == ARG
    assert lib.gr_kv_read(ctypes.byref(c), P, 4, P, P, None, None) == ARG
    assert _attend(cache=c) == ARG


def test_a_cache_past_32_bit_rows_is_refused():
    c = _cache(n_pages=(2 ** 31 // 16) // 8)
    assert _write(cache=c) == UNSUPPORTED and _attend(cache=c) == UNSUPPORTED


@pytest.mark.parametrize("args", [(None, 4, P, P), (P, 0, P, P), (P, -1, P, P), (P, 4, None, P), (P, 4, P, None),
                                  (P, 4, P + 2, P), (P, 4, P, P + 8)])
def test_read_refuses(args):
    assert L.load().gr_kv_read(ctypes.byref(_cache()), *args, None, None) == ARG


def _attend(cache=None, **kw):
    a = dict(q=P, pt=P, stride=8, seq=P, bs=2, K=1, draft=0, add=0, nq=16, chunk=128, splits=1, out=P, ws=None, n_ws=0)
    a.update(kw)
    return L.load().gr_kv8_attention(a["q"], ctypes.byref(cache or _cache()), a["pt"], a["stride"], a["seq"], a["bs"],
                                     a["K"], a["draft"], a["add"], a["nq"], a["chunk"], a["splits"], a["out"], a["ws"],
                                     a["n_ws"], None, None)


@pytest.mark.parametrize("kw", [dict(q=None), dict(q=P + 8), dict(pt=None), dict(stride=0), dict(seq=None), dict(bs=0),
                                dict(K=0), dict(draft=3), dict(draft=-1), dict(nq=12), dict(nq=0), dict(chunk=0),
                                dict(chunk=100), dict(chunk=8224), dict(splits=0), dict(splits=129, ws=P, n_ws=1 << 40),
                                dict(splits=2), dict(splits=2, ws=P, n_ws=65536), dict(splits=2, ws=P + 4, n_ws=1 << 30),
                                dict(out=None), dict(out=P + 2), dict(K=33, nq=16, chunk=32)])
def test_attention_refuses(kw):
    assert _attend(**kw) == ARG


@pytest.mark.parametrize("kw", [dict(K=65), dict(bs=2049), dict(stride=2 ** 27), dict(nq=1032)])
def test_attention_says_unsupported(kw):
    assert _attend(**kw) == UNSUPPORTED


def test_attention_leaves_a_bf16_cache_to_bd_attention():
    assert _attend(cache=_cache(format=L.KV_BF16)) == UNSUPPORTED


def _lp(**kw):
    a = dict(x=P, bf=0, ld=100, rows=2, vocab=100, ids=P, t=None, n=5, lp=P, ent=P, rank=P, top=P, tid=P)
    a.update(kw)
    return L.load().gr_token_logprobs(a["x"], a["bf"], a["ld"], a["rows"], a["vocab"], a["ids"], a["t"], a["n"], a["lp"],
                                      a["ent"], a["rank"], a["top"], a["tid"], None, None)


@pytest.mark.parametrize("kw", [dict(x=None), dict(x=P + 2), dict(bf=1, x=P + 1), dict(ld=99), dict(rows=0),
                                dict(vocab=0), dict(ids=None), dict(n=-1), dict(n=65), dict(vocab=4, n=5), dict(lp=None),
                                dict(ent=None), dict(rank=None), dict(top=None), dict(tid=None)])
def test_logprobs_refuses(kw):
    assert _lp(**kw) == ARG


@pytest.mark.parametrize("bs", [1, 2, 7, 64, 500])
@pytest.mark.parametrize("max_len", [1, 31, 32, 129, 4129, 131072, 2 ** 20])
@pytest.mark.parametrize("heads", [(16, 8), (5, 1), (32, 8)])
def test_plan_covers_the_longest_request(bs, max_len, heads):
    chunk, splits = L.kv8_attention_split(bs, 1, max_len, *heads)
    assert chunk % 32 == 0 and 1 <= splits <= 128 and chunk * splits >= max_len > chunk * (splits - 1)
    assert L.kv8_attention_workspace_bytes(bs, 1, *heads, splits) >= 65536 + bs * heads[0] * splits * 520


def test_plan_refuses():
    lib, out = L.load(), (ctypes.c_int32 * 2)()
    for a in [(1, 1, 2 ** 20 + 1, 16, 8), (0, 1, 9, 16, 8), (1, 0, 9, 16, 8), (1, 1, 0, 16, 8), (1, 1, 9, 15, 8), (1, 1, 9, 16, 0)]:
        assert lib.gr_kv8_attention_plan(*a, out) == ARG
    assert lib.gr_kv8_attention_plan(1, 1, 9, 16, 8, None) == ARG
    assert L.kv8_attention_workspace_bytes(1, 1, 15, 8, 1) == 0


def test_plan_of_too_many_rows():
    """Row counts past the kernel's 128, and past 32 bits."""
    lib, out = L.load(), (ctypes.c_int32 * 2)()
    for K, nq, nkv in [(65, 16, 8), (2 ** 31 - 1, 16, 8), (2 ** 31 - 1, 2 ** 31 - 1, 1), (1, 129, 1)]:
        assert lib.gr_kv8_attention_plan(1, K, 4096, nq, nkv, out) == UNSUPPORTED
        assert L.kv8_attention_workspace_bytes(1, K, nq, nkv, 4) == 0
    assert lib.gr_kv8_attention_plan(2 ** 31 - 1, 1, 2 ** 20, 2 ** 31 - 1, 2 ** 31 - 1, out) == UNSUPPORTED
    assert L.kv8_attention_workspace_bytes(2 ** 31 - 1, 1, 8, 8, 4) == L.kv8_attention_workspace_bytes(1, 1, 8, 8, 129) == 0


def test_wrappers_want_cuda_tensors():
    k = torch.zeros((2, 1, 16, 128), dtype=torch.int8)
    e = torch.zeros((2, 1, 16), dtype=torch.int8)
    with pytest.raises(RuntimeError, match="CUDA"):
        L.kv_cache(k, k, e, e)
    with pytest.raises(RuntimeError, match="no cache format"):
        L.kv_cache(k.float(), k.float())
    x = torch.zeros((2, 8))
    with pytest.raises(RuntimeError, match="CUDA"):
        L.token_logprobs(x, torch.zeros(2, dtype=torch.int64), x[:, 0], x[:, 0], torch.zeros(2, dtype=torch.int32))


def test_oracle_grid_is_torch_s_e4m3():
    every = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    assert torch.equal(every, R.grid("e4m3"))
    x = torch.randn(4096, dtype=torch.float32, generator=torch.Generator().manual_seed(1)) * 40
    assert torch.equal(R.nearest(x.double(), "e4m3"), x.to(torch.float8_e4m3fn).double())
    mid = (every[1:] + every[:-1]) / 2  # ties
    assert torch.equal(R.nearest(mid, "e4m3"), mid.float().to(torch.float8_e4m3fn).double())


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_oracle_exponent(fmt):
    top = R.TOP[fmt]
    rows = torch.zeros((5, 128), dtype=torch.float64)
    rows[1, 3], rows[2, 3], rows[3, 3], rows[4, 3] = top, top * (1 + 2 ** -40), -top * 2.0 ** 60, float("inf")
    codes, e = R.quantise(rows, fmt)
    assert e.tolist() == [-40, 0, 1, 40, -128]
    assert codes[3, 3] == -top and torch.isnan(R.values(codes, e)[4]).all()
