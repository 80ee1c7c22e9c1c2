"""Token log probabilities of many and of long rows on a B200: every CTA size (128 threads above four rows an SM, 256 above two, 512
and clusters below), threads with more batches than cells, the fetch ahead of a later row, rows with few or no tokens among
them; against the 64-bit oracle (run on the GPU in float64).

Bounds.  R is a fp32 sum of terms e = 2^d.  d = (x - ref) k has three roundings (k's among them) and moves with the reference
once: for |d| <= 64 that is 4 x 64 ln 2 x 2^-24 of e.  A thread adds its n terms in two sums of n / 2, then a few, then 5 + 4
steps of a tree and the 16 of a join: (n / 2 + 40) 2^-24.  So R is off by rel R, rel = (n / 2 + 240) 2^-24 (ex2's 2^-22 and the
tail of smaller terms included), log1p(R) by rel R / (1 + R) <= rel log1p(R), W by (rel + 2^-22) W, and H = log1p(R) -
W / (1 + R), both terms >= 0, by (3 rel + 2^-21) H.  log p = d - log1p(R), both <= 0, has roundings of its own: 2^-21 of it."""
import pytest
import torch

from gravityocr_b200 import _lib as L
from oracle import kv8_ref as R
from test_gpu_logprobs import DEV, _call

pytestmark = pytest.mark.gpu


def _threads(rows):
    sms = L.num_sms()
    return 128 if rows > 4 * sms else (256 if rows > 2 * sms else 512)


def _rows(rows, vocab, dtype, seed, pad=0):
    """Random rows with a few loud tokens; every kind of special row in turn among them."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn((rows, vocab + pad), generator=g, device=DEV) * 3
    x += torch.where(torch.rand(x.shape, generator=g, device=DEV) < 3.0 / vocab, 8.0, 0.0)
    ids = torch.randint(0, vocab, (rows,), generator=g, device=DEV)
    i = torch.arange(vocab + pad, device=DEV)
    low = float(torch.finfo(dtype).min)
    for r in range(0, rows, 13):
        kind = r // 13 % 12
        if kind == 0:
            x[r] = 2.5                                         # every token equal
        elif kind == 1:
            x[r] = (i % 3).float()                             # few values, many ties
        elif kind == 2:
            x[r] = (i // 2048) + (i % 4) / 8
        elif kind == 3:
            x[r, ::4] = float("-inf")
        elif kind == 4:
            x[r, vocab // 5:] = float("-inf")
        elif kind == 5:                                        # three tokens left
            keep = x[r, ids[r]].clone()
            x[r] = float("-inf")
            x[r, [1, vocab // 2, vocab - 1]] = torch.tensor([1.0, 1.0, 0.5], device=DEV)
            x[r, ids[r]] = keep
        elif kind == 6:                                        # one
            x[r] = float("-inf")
            x[r, vocab // 3] = -7.0
        elif kind == 7:
            x[r, 1::2] = low
        elif kind == 8:
            x[r] = low
        elif kind == 9:
            x[r] = float("-inf")
        elif kind == 10:
            x[r, vocab - 2] = float("nan")
        else:
            x[r, vocab // 7] = float("inf")
    return x.to(dtype)[:, :vocab], ids


def _check(x, ids, n, temperature=None):
    rows, vocab = x.shape
    st = torch.zeros((1,), dtype=torch.int32, device=DEV)
    lp, ent, rank, top, tid = _call(x, ids, n, temperature, st)
    y = x.float()
    has = ~torch.isnan(y).any(1) & (y.amax(1) > -float("inf")) & (y.amax(1) < float("inf"))
    del y
    assert int(st) == (0 if bool(has.all()) else L.GR_ERR_NO_TOKEN)
    none = ~has
    assert torch.isnan(lp[none]).all() and torch.isnan(ent[none]).all() and (rank[none] == 0).all()
    assert torch.isnan(top[none]).all() and (tid[none] == -1).all()
    rel = ((vocab / _threads(rows) + 32) / 2 + 240) * 2.0 ** -24
    kept = torch.nonzero(has)[:, 0]
    for part in kept.split(200):
        t = None if temperature is None else temperature.to(DEV)[part]
        wlp, went, wrank, wtop, wtid = R.logprobs(x[part], ids[part], t, n)
        assert torch.equal(rank[part].long(), wrank) and torch.equal(tid[part].long(), wtid)
        r = torch.expm1(-wtop[:, 0])
        slack = rel * r / (1 + r)
        for got, want, s in ((lp[part], wlp, slack), (top[part], wtop, slack[:, None])):
            # what fp32 does not hold rounds to it: -inf, and numbers below its lowest (3.4e38 / T for a T below one) to -inf
            got, held = got.double(), want.float().double()
            assert ((got == held) | ((got - want).abs() <= s + 2.0 ** -21 * want.abs())).all()
        assert ((ent[part].double() - went).abs() <= (3 * rel + 2.0 ** -21) * went + 1e-30).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,n,pad", [
    (1, 59392, 20, 0), (64, 59392, 20, 0), (150, 59392, 20, 3),                    # clusters, 512 threads
    (200, 300001, 64, 0),                                                          # cells taken again
    (300, 59392, 64, 0), (400, 59392, 20, 1), (592, 9000, 33, 8),                  # 256 threads
    (593, 59392, 20, 0), (600, 59392, 64, 1), (700, 3001, 20, 0), (1088, 59392, 20, 0), (1200, 59392, 64, 5),   # 128 threads
    (1300, 131, 64, 2), (2500, 64, 64, 0), (1190, 2049, 1, 0)])
def test_rows(rows, vocab, n, pad, dtype):
    x, ids = _rows(rows, vocab, dtype, rows + vocab, pad)
    _check(x, ids, n)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(610, 131072), (310, 131072), (1088, 20000)])
def test_rows_at_temperatures(rows, vocab, dtype):
    x, ids = _rows(rows, vocab, dtype, 7)
    _check(x, ids, 20, 0.5 + 2.0 * torch.rand((rows,), generator=torch.Generator().manual_seed(1)))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows", [1, 8, 64, 150, 310, 600, 1088])
@pytest.mark.parametrize("legal", [1, 3, 19, 20, 21])
def test_fewer_tokens_than_alternatives(rows, legal, dtype):
    """A grammar that leaves `legal` of 59,392 tokens, n = 20: the rest are the lowest masked ids."""
    vocab = 59392
    g = torch.Generator(device=DEV).manual_seed(legal)
    x = torch.full((rows, vocab), float("-inf"), device=DEV)
    at = torch.randint(0, vocab, (rows, legal), generator=g, device=DEV)
    x.scatter_(1, at, torch.randint(-8, 8, (rows, legal), generator=g, device=DEV) / 4)
    _check(x.to(dtype), at[:, 0].contiguous(), 20)


@pytest.mark.parametrize("rows", [600, 1088])
def test_a_row_does_not_depend_on_its_batch(rows):
    """The 128-thread rows of a batch, from any place in it."""
    x, ids = _rows(rows, 59392, torch.float32, 3)
    a = _call(x, ids, 20)
    order = torch.randperm(rows, generator=torch.Generator().manual_seed(2)).to(DEV)
    b = _call(x[order].contiguous(), ids[order].contiguous(), 20)
    for p, q in zip(a, b):
        assert torch.equal(p[order].nan_to_num(5.0), q.nan_to_num(5.0))
