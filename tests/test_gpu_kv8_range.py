"""8-bit cache attention at the ends of the exponents' range: tiles whose weights 2^(score + exponent) lie far apart, in one chunk
and across splits, against the 64-bit oracle (scores and bounds as in test_gpu_kv8)."""
import math

import pytest
import torch

from gravityocr_b200 import _lib as L
from oracle import kv8_ref as R
from test_gpu_kv8 import DEV, DT, _attend, _attn_case, _check_attention, _status

pytestmark = pytest.mark.gpu


def _case(fmt, tokens, score):
    """One request of len(tokens) tokens, one head.  tokens: (0 or 1, e): the key of score 0 or of about `score` (base 2), and a
    value row of 0.8 top 2^e."""
    n = len(tokens)
    c = _attn_case(fmt, [n - 1], 1, 1, 1, spread=0.0)
    k, v, ke, ve = c["cache"]
    q = torch.zeros((1, 128))
    q[0, 0] = score * math.sqrt(128) / (8 * math.log2(math.e))
    c["q"] = q.bfloat16()
    slots = c["slots"][0]
    pages = k.shape[0]
    rows_k, rows_v = (torch.zeros((pages * 16, 128), dtype=torch.float64) for _ in range(2))
    loud = torch.tensor([t[0] for t in tokens], dtype=torch.float64)
    e = torch.tensor([t[1] for t in tokens], dtype=torch.float64)
    rows_k[slots, 0] = 8 * loud
    # a row's values differ by dimension (the sign and the size), its largest decides the exponent
    shape = torch.linspace(-1, 1, 128, dtype=torch.float64)
    rows_v[slots] = (0.8 * R.TOP[fmt] * 2.0 ** e)[:, None] * shape
    for rows, codes, exps, name in ((rows_k, k, ke, "k"), (rows_v, v, ve, "v")):
        qc, ex = R.quantise(rows.view(pages, 1, 16, 128), fmt)
        codes.copy_(qc.float().to(DT[fmt]))
        exps.copy_(ex.to(torch.int8))
        c[name] = R.values(qc, ex).transpose(1, 2).flatten(0, 1)
    assert ve.cpu().transpose(1, 2).flatten()[slots].tolist() == e.int().tolist()
    return c


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("score", [60, 87, 103, 130])
@pytest.mark.parametrize("chunk", [8192, 2048])
def test_a_sum_of_thousands_of_quiet_rows(fmt, score, chunk):
    """A first tile of ordinary rows, then thousands of tokens with all the weight and the quietest values (2^-ev = 2^40 each in
    the softmax sum): the sum stays finite, the output is their mean."""
    c = _case(fmt, [(0, 0)] * 128 + [(1, -40)] * 7000, score)
    st = _status()
    out = _attend(c, chunk=chunk, status=st)
    assert int(st) == 0
    _check_attention(c, out)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("score", [70, 85, 87, 100, 127, 200])
@pytest.mark.parametrize("chunk", [8192, 128, 256])
@pytest.mark.parametrize("order", ["quiet first", "loud first"])
def test_equal_scores_whose_values_are_80_binades_apart(fmt, score, chunk, order):
    """Two tokens of the same score, in tiles of their own behind one of score 0: their weights 2^(score + e) are 2^80 apart, the
    softmax has them equal.  One chunk (the sums' reference rises between them), a split each, and a split that holds the
    quiet one beside the first tile."""
    quiet = [(1, -40)] + [(0, -40)] * 127
    loud = [(1, 40)] + [(0, 0)] * 127
    first = [(0, 0)] * 128
    tiles = [first, quiet, loud] if order == "quiet first" else [loud, first, quiet]
    c = _case(fmt, [t for tile in tiles for t in tile], score)
    st = _status()
    out = _attend(c, chunk=chunk, status=st)
    assert int(st) == 0
    _check_attention(c, out)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("chunk", [8192, 384])
def test_many_quiet_tokens_behind_a_raise(fmt, chunk):
    """A thousand quiet tokens 39 binades below one loud weight hold the softmax sum between them, before and after it."""
    quiet, loud = [(1, -40)] * 512, [(1, 40)] + [(0, 0)] * 127
    for tokens in ([(0, 0)] * 128 + quiet + loud + quiet, loud + quiet + [(0, 0)] * 300 + quiet):
        c = _case(fmt, tokens, 87)
        _check_attention(c, _attend(c, chunk=chunk))


@pytest.mark.parametrize("splits", [1, 2])
def test_more_row_blocks_than_16384(splits):
    """600 requests' prompt chunks of 64 rows: 4,800 (request, head) pairs of four row blocks, each with a ticket of its own."""
    bs, K, nq, nkv = 600, 64, 16, 8
    c = _attn_case("int8", [0, 60, 17, 1, 40, 5, 33, 58], K, nq, nkv)    # eight different ones, over and over
    g = torch.Generator().manual_seed(1)
    lens, slots = c["lens"] * 75, c["slots"] * 75
    c.update(bs=bs, lens=lens, slots=slots, pt=c["pt"].repeat(75, 1),
             q=torch.randn((bs * K, nq * 128), generator=g).bfloat16())
    chunk = 128 // splits
    ws = torch.zeros((L.kv8_attention_workspace_bytes(bs, K, nq, nkv, splits),), dtype=torch.uint8, device=DEV)
    st = _status()
    # a small call first: its partial results lie behind the tickets, whatever the shape
    small = dict(c, pt=c["pt"][:8].contiguous(), q=c["q"][: 8 * K], lens=lens[:8], slots=slots[:8], bs=8)
    _check_attention(small, _attend(small, chunk=32, splits=4, ws=ws, status=st))
    out = _attend(c, chunk=chunk, splits=splits, ws=ws, status=st)
    again = _attend(c, chunk=chunk, splits=splits, ws=ws, status=st)
    assert int(st) == 0 and torch.equal(out, again)
    tickets = 4 * bs * nkv * 4
    assert int(ws[:tickets].sum()) == 0
    for b in (0, 1, 300, 555, 599):
        one = dict(c, pt=c["pt"][b: b + 1].contiguous(), q=c["q"][b * K: (b + 1) * K], lens=[lens[b]], bs=1, slots=slots[b: b + 1])
        _check_attention(one, out[b * K: (b + 1) * K])
