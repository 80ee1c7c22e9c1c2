"""Token log probabilities on a B200 against the 64-bit oracle: ranks and ids have to be equal, the numbers stay within
bounds derived from the arithmetic."""
import math

import pytest
import torch

from gravityocr_b200 import _lib as L
from oracle import kv8_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _call(logits, ids, n, temperature=None, status=None, stream=None):
    rows = logits.shape[0]
    o = dict(lp=torch.full((rows,), 9.0, device=DEV), ent=torch.full((rows,), 9.0, device=DEV),
             rank=torch.full((rows,), 9, dtype=torch.int32, device=DEV))
    top = torch.full((rows, n), 9.0, device=DEV) if n else None
    tid = torch.full((rows, n), 9, dtype=torch.int32, device=DEV) if n else None
    L.token_logprobs(logits, ids.to(DEV), o["lp"], o["ent"], o["rank"], top_logprob=top, top_ids=tid,
                     temperature=None if temperature is None else temperature.to(DEV), status=status, stream=stream)
    return o["lp"], o["ent"], o["rank"], top, tid


def _check(logits, ids, n, temperature=None):
    st = torch.zeros((1,), dtype=torch.int32, device=DEV)
    lp, ent, rank, top, tid = _call(logits, ids, n, temperature, st)
    assert int(st) == 0
    wlp, went, wrank, wtop, wtid = R.logprobs(logits.cpu(), ids, temperature, max(n, 1))
    assert torch.equal(rank.cpu().long(), wrank)
    # log1p(R): R's relative error is that of its terms (2^-22, and |d| <= 40 in base 2 times 2^-23 where they matter) and of
    # a fp32 sum of at most 256 terms a thread and 16 joins: below 2^-16 R; the rest are roundings of the result
    r = torch.expm1(-wtop[:, 0])
    slack = 2.0 ** -16 * r / (1 + r)
    lp = lp.double().cpu()
    assert ((lp == wlp) | ((lp - wlp).abs() <= slack + 2.0 ** -21 * wlp.abs())).all()   # (-inf equals -inf)
    # H = log1p(R) - W / (1 + R): two terms >= 0, W's terms with the same errors and one more product
    assert ((ent.double().cpu() - went).abs() <= 2.0 ** -14 * went + 1e-30).all()
    if n:
        assert torch.equal(tid.cpu().long(), wtid)
        fin = torch.isfinite(wtop)
        err = (top.double().cpu() - wtop).abs()
        assert (err[fin] <= (slack[:, None] + 2.0 ** -21 * wtop.abs())[fin]).all()
        assert torch.equal(top.cpu()[~fin].double(), wtop[~fin])


def _logits(rows, vocab, dtype, seed, pad=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((rows, vocab + pad), generator=g) * 3
    x[:, : vocab] += torch.where(torch.rand((rows, vocab), generator=g) < 3.0 / vocab, 8.0, 0.0)
    return x.to(dtype).to(DEV)[:, :vocab], torch.randint(0, vocab, (rows,), generator=g)


SIZES = [(1, 1), (1, 2), (3, 5), (2, 7), (5, 63), (4, 1000), (3, 4099), (1, 59392), (2, 59392), (9, 59391), (300, 2050),
         (40, 8192), (2, 131072), (1, 600001)]


@pytest.mark.parametrize("rows,vocab", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sizes(rows, vocab, dtype):
    x, ids = _logits(rows, vocab, dtype, rows * vocab)
    _check(x, ids, min(vocab, 20))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("pad", [1, 3, 4, 8])
def test_row_strides_and_unaligned_rows(dtype, pad):
    x, ids = _logits(7, 1001, dtype, pad, pad)
    _check(x, ids, 5)
    _check(x[:, 1:], ids.clamp_max(999), 5)


@pytest.mark.parametrize("n", [0, 1, 2, 31, 33, 64])
@pytest.mark.parametrize("rows", [1, 30, 200])
def test_counts_of_alternatives(n, rows):
    x, ids = _logits(rows, 5000, torch.float32, n)
    _check(x, ids, n)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_temperature(dtype):
    x, ids = _logits(6, 59392, dtype, 1)
    _check(x, ids, 20, torch.tensor([0.01, 0.3, 0.7, 1.0, 1.7, 100.0]))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [64, 5000, 59392])
def test_ties_and_orders(dtype, vocab):
    """Equal rows, few distinct values, rising and falling rows, +0 / -0, the best ones side by side or far apart."""
    g = torch.Generator().manual_seed(vocab)
    i = torch.arange(vocab, dtype=torch.float32)
    best_near, best_far = torch.zeros(vocab), torch.zeros(vocab)
    best_near[: 64] = 5.0
    best_far[:: max(1, vocab // 64)] = 5.0
    x = torch.stack([torch.full((vocab,), 2.5), torch.randint(0, 3, (vocab,), generator=g).float(), i / 64, -i / 64,
                     torch.where(i % 2 == 0, 0.0, -0.0), best_near, best_far, -(i % 512),
                     (i // 2048) + (i % 4) / 8]).to(dtype).to(DEV)
    for k in (0, vocab // 2, vocab - 1):
        _check(x, torch.full((x.shape[0],), k), 64)


def test_many_candidates():
    """The elements above the first bound overflow the candidate list: a few threads hold every large logit."""
    vocab = 59392
    for stride, lanes in ((2048, 32), (4096, 64), (2048, 160)):
        x = torch.zeros((2, vocab))
        i = torch.arange(vocab)
        g = torch.Generator().manual_seed(lanes)
        hot = (i % stride) < lanes
        x[0, hot] = 10 + torch.rand(int(hot.sum()), generator=g)
        x[1, hot] = 10 + torch.arange(int(hot.sum())) / 4096
        for dtype in (torch.float32, torch.bfloat16):
            _check(x.to(dtype).to(DEV), torch.tensor([3, vocab - 1]), 64)


@pytest.mark.parametrize("vocab", [40, 59392])
def test_masked_tokens(vocab):
    """-inf logits: some, all but one, all but a few, in the asked token's place; runs that fill whole vectors."""
    x, ids = _logits(5, vocab, torch.float32, 4)
    x[0, vocab // 3:] = float("-inf")
    x[1, :] = float("-inf")
    x[1, vocab // 2] = -3.0
    x[2, :] = float("-inf")
    x[2, [1, vocab // 2, vocab - 1]] = torch.tensor([1.0, 2.0, 1.0], device=DEV)
    x[3, ids[3]] = float("-inf")
    x[4, ::2] = float("-inf")
    lp, ent, rank, top, tid = _call(x, ids, 8)
    w = R.logprobs(x.cpu(), ids, None, 8)
    assert torch.equal(rank.cpu().long(), w[2]) and torch.equal(tid.cpu().long(), w[4])
    assert float(lp[3]) == float("-inf") and float(ent[1]) == 0.0 and float(top[1, 0]) == 0.0
    assert (top[1, 1:] == float("-inf")).all()
    fin = torch.isfinite(w[0])
    assert ((lp.double().cpu() - w[0])[fin].abs() <= 2.0 ** -16 + 2.0 ** -21 * w[0][fin].abs()).all()
    assert torch.equal(lp.cpu()[~fin].double(), w[0][~fin])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab,rows", [(100, 2), (59392, 3), (59392, 200)])
def test_masks_of_the_lowest_value(dtype, vocab, rows):
    """Masks of the type's lowest value: some tokens, all of them (a uniform row), mixed with -inf, all but very low ones."""
    low = torch.finfo(dtype).min
    x, ids = _logits(rows, vocab, dtype, 5)
    x[0, ::2] = low
    x[0, 1] = float("-inf")
    x[1, :] = low
    _check(x, ids, 10)
    x[0, :] = float("-inf")
    x[0, 3:9] = low
    x[1, :] = low
    x[1, vocab // 2:] = -3e30
    lp, ent, rank, top, tid = _call(x, torch.full_like(ids, 4), 10)
    assert abs(float(ent[0]) - math.log(6)) < 1e-6 and abs(float(lp[0]) + math.log(6)) < 1e-6 and int(rank[0]) == 2
    assert tid[0].tolist() == [3, 4, 5, 6, 7, 8, 0, 1, 2, 9]
    n = vocab - vocab // 2
    assert abs(float(ent[1]) - math.log(n)) < 1e-5 and float(lp[1]) < -1e38 and int(rank[1]) == n + 5
    assert tid[1].tolist() == list(range(vocab // 2, vocab // 2 + 10))


def test_peaked_rows_keep_their_digits():
    """log p of a near-certain token is -R, far below fp32's step at 1."""
    x = torch.full((4, 59392), -60.0, device=DEV)
    x[0, 5], x[1, 5], x[2, 5], x[3, 5] = 0.0, -20.0, -40.0, -45.0
    x[3, 59391] = -45.0
    _check(x, torch.full((4,), 5), 3)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_without_a_distribution(dtype):
    x, ids = _logits(6, 3001, dtype, 8)
    x[0, 100] = float("nan")
    x[1, 2999] = float("inf")
    x[2, :] = float("-inf")
    x[3, :] = float("nan")
    st = torch.zeros((1,), dtype=torch.int32, device=DEV)
    lp, ent, rank, top, tid = _call(x, ids, 4, status=st)
    assert int(st) == L.GR_ERR_NO_TOKEN
    for r in range(4):
        assert torch.isnan(lp[r]) and torch.isnan(ent[r]) and int(rank[r]) == 0
        assert torch.isnan(top[r]).all() and (tid[r] == -1).all()
    _check(x[4:], ids[4:], 4)
    w = R.logprobs(x[4:].cpu(), ids[4:], None, 4)
    assert torch.equal(tid[4:].cpu().long(), w[4])


def test_ids():
    x, ids = _logits(3, 1000, torch.float32, 2)
    st = torch.zeros((1,), dtype=torch.int32, device=DEV)
    lp, ent, rank, top, tid = _call(x, torch.tensor([-1, 7, -1]), 3, status=st)
    assert int(st) == 0 and torch.isnan(lp[[0, 2]]).all() and rank.tolist()[0] == 0 and float(lp[1]) < 0
    assert torch.isfinite(ent).all() and torch.isfinite(top).all()
    for bad in (1000, -2, 2 ** 40):
        st.zero_()
        lp, _, rank, top, _ = _call(x, torch.tensor([1, bad, 2]), 3, status=st)
        assert int(st) == 5 and torch.isnan(lp[1]) and int(rank[1]) == 0 and torch.isfinite(lp[[0, 2]]).all()
        assert torch.isfinite(top).all()


def test_bad_temperature():
    x, ids = _logits(4, 1000, torch.float32, 2)
    st = torch.zeros((1,), dtype=torch.int32, device=DEV)
    lp, _, rank, _, tid = _call(x, ids, 3, torch.tensor([0.0, -1.0, float("nan"), 1.0]), status=st)
    assert int(st) == 1 and torch.isnan(lp[:3]).all() and float(lp[3]) <= 0 and (tid[:3] == -1).all()


def test_streams_and_graphs():
    """A captured call replays over new logits, on a stream of its own, and equals the eager call."""
    x, ids = _logits(130, 59392, torch.float32, 3)
    buf, idb = torch.zeros_like(x), ids.to(DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            pass_out = _call(buf, idb, 20)
        buf.copy_(x)
        g.replay()
    s.synchronize()
    for a, b in zip(pass_out, _call(x, ids, 20)):
        assert torch.equal(a, b)


def test_wrapper_refuses():
    x, ids = _logits(3, 100, torch.float32, 2)
    f, r = torch.zeros(3, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV)
    idd = ids.to(DEV)
    with pytest.raises(RuntimeError, match="unit column stride"):
        L.token_logprobs(x.t(), idd, f, f, r)
    with pytest.raises(RuntimeError, match="logits must"):
        L.token_logprobs(x.half(), idd, f, f, r)
    with pytest.raises(RuntimeError, match="come together"):
        L.token_logprobs(x, idd, f, f, r, top_ids=torch.zeros((3, 2), dtype=torch.int32, device=DEV))
    with pytest.raises(RuntimeError, match="ids holds"):
        L.token_logprobs(x, idd[:2], f, f, r)
    with pytest.raises(RuntimeError, match="invalid argument"):
        L.token_logprobs(x, idd, f, f, r, top_logprob=torch.zeros((3, 65), device=DEV),
                         top_ids=torch.zeros((3, 65), dtype=torch.int32, device=DEV))
