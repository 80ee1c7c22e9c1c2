"""The engine's own 8-bit attention on a B200: what the last layer of a prefill chunk, of a draft and of a verify forward computed,
from the engine's query rows over the cache as it lies, against the 64-bit oracle (masks, lengths, page tables, batches), and
the rows that the last layer wrote, code by code."""
import pytest
import torch

from oracle import kv8_ref as R
from test_gpu_kv8 import _check_attention
from test_gpu_kv8_round import K, _setup

pytestmark = pytest.mark.gpu


def _case(eng, rb, lens, rows):
    """The last layer's attention of `rows` new rows a request behind `lens` tokens, as test_gpu_kv8 describes one."""
    cfg, pool = eng.cfg, eng.pool
    bs = len(lens)
    held = []
    for codes, exps in ((pool.k[-1], pool.k_exp[-1]), (pool.v[-1], pool.v_exp[-1])):
        c = codes.cpu()
        c = c.float() if c.dtype == torch.float8_e4m3fn else c
        held.append(R.values(c, exps.cpu()).transpose(1, 2).flatten(0, 1))
    pt = rb.page_table.cpu().long()
    slots = []
    for b in range(bs):
        t = torch.arange(lens[b] + rows)
        slots.append(pt[b][t // 16] * 16 + t % 16)
    return dict(cache=(pool.k[-1],), k=held[0], v=held[1], slots=slots, q=eng.q[: bs * rows].cpu(), lens=lens, K=rows,
                nq=cfg.n_q_heads, nkv=cfg.n_kv_heads, bs=bs)


def _check_rows_written(eng, c, rows, fmt):
    """The new rows' codes are the rotation of the engine's projected rows, rounded once."""
    cfg = eng.cfg
    for b in range(c["bs"]):
        y = eng.qkv[b * rows: (b + 1) * rows].cpu().double().view(rows, -1, 128)
        pos = torch.arange(c["lens"][b], c["lens"][b] + rows)
        k = R.norm_rotate(y[:, cfg.n_q_heads: cfg.n_q_heads + cfg.n_kv_heads], None, 0.0, R.angles(eng.w.inv_freq.cpu(), pos), False)
        v = y[:, cfg.n_q_heads + cfg.n_kv_heads:]
        new = c["slots"][b][c["lens"][b]:]
        for held, ref in ((c["k"], k), (c["v"], v)):
            assert torch.equal(held[new], R.values(*R.quantise(ref, fmt)))


@pytest.mark.parametrize("fmt,dtype", [("int8", torch.int8), ("e4m3", torch.float8_e4m3fn)])
def test_prefill_draft_and_verify(fmt, dtype):
    cfg, w32, reqs, eng, rb, cap = _setup(dtype, n_image=90, n_prompt=30, bs=3)
    eng.prefill(rb, [r[0][: 120 - 37 * b] for b, r in enumerate(reqs)], [r[1][: 120 - 37 * b] for b, r in enumerate(reqs)])
    torch.cuda.synchronize()
    # the last chunk: rows 64-127 of the requests that are longer than 64 (the third has 46)
    c = _case(eng, rb, [64, 64], 64)
    _check_attention(c, eng.attn[: 2 * 64])
    for r in range(3):
        lens = rb.seq_lens.tolist()
        eng.draft_launch(rb)
        torch.cuda.synchronize()
        c = _case(eng, rb, lens, K)
        _check_attention(c, eng.attn[: 3 * K], draft=1)
        _check_rows_written(eng, c, K, fmt)
        eng.verify_launch(rb)
        torch.cuda.synchronize()
        c = _case(eng, rb, [n + 1 for n in lens], K)
        _check_attention(c, eng.attn[: 3 * K])
        _check_rows_written(eng, c, K, fmt)
    eng.check_status(rb)
