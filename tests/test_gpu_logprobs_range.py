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
