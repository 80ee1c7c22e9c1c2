"""The plan, the workspace size and the call of the 8-bit attention take the same shapes.  (No call here is accepted: each has a
flaw that is looked at after its shape.)"""
import ctypes

import pytest

from gravityocr_b200 import _lib as L
from test_kv8_host import ARG, P, UNSUPPORTED, _attend

PAIRS = [1, 4095, 4096, 4097, 4800, 5461, 5462, 8191, 8192, 8193, 16383, 16384, 16385]


def _entries(bs, K, nq, nkv):
    """What each entry says: supported or not."""
    from test_kv8_host import _cache
    out = (ctypes.c_int32 * 2)()
    plan = L.load().gr_kv8_attention_plan(bs, K, 4096, nq, nkv, out)
    size = L.kv8_attention_workspace_bytes(bs, K, nq, nkv, 2)
    cache = _cache(n_kv_heads=nkv)
    split = _attend(cache=cache, bs=bs, K=K, nq=nq, chunk=2048, splits=2)       # no workspace
    assert plan in (0, UNSUPPORTED) and split in (ARG, UNSUPPORTED)
    says = [plan == 0, size != 0, split == ARG]
    if K > 32:
        whole = _attend(cache=cache, bs=bs, K=K, nq=nq, chunk=32, splits=1)     # a chunk that does not hold the window
        assert whole in (ARG, UNSUPPORTED)
        says.append(whole == ARG)
    return says


@pytest.mark.parametrize("rows", [1, 33, 34, 40, 41, 80, 81, 120, 121, 128, 129])
@pytest.mark.parametrize("nkv", [1, 8])
def test_the_three_entries_agree(rows, nkv):
    for pairs in PAIRS:
        if pairs % nkv == 0:
            want = rows <= 128 and pairs <= 16384
            assert _entries(pairs // nkv, rows, nkv, nkv) == [want] * (4 if rows > 32 else 3), (pairs, rows)
            assert _entries(pairs // nkv, 1, rows * nkv, nkv) == [want] * 3, (pairs, rows)


def test_the_prefill_of_600_requests_is_planned_and_taken():
    assert all(_entries(600, 64, 16, 8))


@pytest.mark.parametrize("bs,K", [(600, 64), (2048, 64), (1, 64), (64, 17)])
def test_the_workspace_holds_every_ticket_and_partial(bs, K):
    blocks = -(-2 * K // 40)
    assert L.kv8_attention_workspace_bytes(bs, K, 16, 8, 3) >= 4 * max(16384, bs * 8 * blocks) + bs * 8 * 3 * 2 * K * 520
