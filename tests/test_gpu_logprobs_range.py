"""Token log probabilities at the ends of the numbers' range: temperatures down to the smallest normal number and infinite ones, logits
far apart; against the 64-bit oracle with the bounds of test_gpu_logprobs."""
import math

import pytest
import torch

from gravityocr_b200 import _lib as L
from oracle import kv8_ref as R
from test_gpu_logprobs import DEV, _call, _check, _logits

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,vocab", [(1, 59392), (7, 1001), (200, 59392), (400, 59392), (650, 40000)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_entropy_of_a_row_with_one_far_token(rows, vocab, dtype):
    """Threads whose sums are large (logits up to 24 binades above their first ones), and one token so far above them that their
    weight is 0: the sums must not pass fp32 on the way."""
    x = torch.full((rows, vocab), 16.5)
    x[:, : vocab // 2] = 0.0
    x[:, vocab // 3] = 3e37
    _check(x.to(dtype).to(DEV), torch.full((rows,), vocab // 3), 5)
    x[:, vocab // 3] = 16.5
    x[:, vocab - 1] = 2e31
    _check(x.to(dtype).to(DEV), torch.full((rows,), vocab - 1), 5)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(5, 59392), (605, 3001)])
def test_temperatures_of_any_size(dtype, rows, vocab):
    """From the smallest normal number to the largest, each over logits of its size."""
    some = torch.tensor([2.0 ** -126, 1e-30, 1e-5, 1e30, 3e38])
    t = some[torch.arange(rows) % 5]
    x, ids = _logits(rows, vocab, torch.float32, 3)
    x = (x.cpu() * t.clamp_max(1e37)[:, None]).to(dtype).to(DEV)
    _check(x, ids, 5, t)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab", [(2, 59392), (310, 4000), (605, 3001)])
def test_infinite_temperature(dtype, rows, vocab):
    """Uniform over the tokens that are not masked; ranks and best tokens by logit as ever."""
    x, ids = _logits(rows, vocab, dtype, 4)
    x[:, 1::3] = float("-inf")
    ids = ids // 3 * 3
    ids[-1] = 1
    n = vocab - len(range(1, vocab, 3))
    st = torch.zeros((1,), dtype=torch.int32, device=DEV)
    lp, ent, rank, top, tid = _call(x, ids, 7, torch.full((rows,), float("inf")), status=st)
    assert int(st) == 0
    w = R.logprobs(x.cpu(), ids, None, 7)
    assert torch.equal(rank.cpu().long(), w[2]) and torch.equal(tid.cpu().long(), w[4])
    # log n: a fp32 sum of ones (exact below 2^24), e^d off by 2^-20 at most, log1p and the roundings of the result
    off = 2.0 ** -18 * math.log(n)
    assert ((lp[:-1].double().cpu() + math.log(n)).abs() <= off).all() and float(lp[-1]) == float("-inf")
    assert ((ent.double().cpu() - math.log(n)).abs() <= off).all()
    assert ((top.double().cpu() + math.log(n)).abs() <= off).all()
    few = torch.full((1, 40), float("-inf"), device=DEV)
    few[0, 3] = 2.0
    lp, ent, rank, top, tid = _call(few, torch.tensor([3]), 3, torch.tensor([float("inf")]))
    assert float(lp) == 0 and float(ent) == 0 and top[0].tolist() == [0.0, -math.inf, -math.inf] and tid[0].tolist() == [3, 0, 1]


def test_temperatures_below_the_normal_numbers_are_refused():
    x, ids = _logits(3, 1000, torch.float32, 2)
    for bad in (1e-39, 1e-45, 0.0, -1e-39):
        st = torch.zeros((1,), dtype=torch.int32, device=DEV)
        lp, ent, rank, top, tid = _call(x, ids, 3, torch.tensor([1.0, bad, 1.0]), status=st)
        assert int(st) == 1 and torch.isnan(lp[1]) and torch.isnan(ent[1]) and int(rank[1]) == 0
        assert torch.isnan(top[1]).all() and (tid[1] == -1).all() and torch.isfinite(lp[[0, 2]]).all()
