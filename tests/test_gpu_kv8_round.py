"""Rounds over an 8-bit K/V cache on a B200: the engine's prefill, draft, verify and commit with ``kv_dtype`` set, against the
fp32 oracle (within the cache's rounding) and against themselves (graphs, batches, lengths)."""
import math

import pytest
import torch

from gravityocr_b200 import _lib as L
from gravityocr_b200.config import small_model
from gravityocr_b200.engine import Engine, PagePool
from gravityocr_b200.weights import grid_positions, prefix_embeddings, random_weights, request_inputs
from oracle import kv8_ref as R
from oracle.decoder_ref import OracleDecoder, SpecState, spec_commit, spec_draft, spec_verify

pytestmark = pytest.mark.gpu
DEV = "cuda"
K = 17
# A cached value is off by half a step: relative to its row's largest, 2^-8 (int8), to itself 2^-4 (e4m3); the independent
# errors of a row's 128 products and of the tokens average, so a logit moves by that at most, relative to the row's
# largest logit, through the two layers.
REL = {torch.int8: 2.0 * 2 ** -8, torch.float8_e4m3fn: 2.0 * 2 ** -4}


def _setup(dtype, n_image=64, n_prompt=16, new=64, bs=1, seed=0):
    cfg = small_model(2)
    w = random_weights(cfg, seed, torch.bfloat16)
    w32 = {k: v.float() for k, v in w.items()}
    reqs = []
    for b in range(bs):
        img, txt = request_inputs(cfg, seed, n_image, n_prompt, b, torch.bfloat16)
        reqs.append((prefix_embeddings(w32, cfg, img, txt),
                     torch.cat([torch.full((n_image,), -1, dtype=torch.int64), txt])))
    cap = n_image + n_prompt + new + 4 * K + 64
    ppr = (cap + 15) // 16
    eng = Engine(cfg, w, max_rows=max(64 * bs, bs * K), n_pages=bs * ppr + 4, kv_dtype=dtype)
    eng.reserve(bs * K)
    rb = eng.new_round_buffers(bs, K, ppr, max_len=cap, avg_len=n_image + n_prompt)
    rb.attn_chunk, rb.attn_splits = 128, int(math.ceil((cap + K + 1) / 128))
    for b in range(bs):
        rb.page_table[b] = torch.tensor(eng.pool.alloc(ppr), dtype=torch.int32, device=DEV)
    return cfg, w32, reqs, eng, rb, cap


def _rows_close(gpu_idx, gpu_top, lg, rel):
    top = lg.amax(-1)
    scale = lg.abs().amax(-1)
    assert ((gpu_top - top).abs() <= rel * scale).all()
    chosen = lg.gather(1, gpu_idx.long()[:, None])[:, 0]
    assert (top - chosen <= rel * scale).all()      # the GPU's token is the oracle's, or within the cache's rounding of it


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
def test_round_against_the_oracle(dtype):
    cfg, w32, reqs, eng, rb, cap = _setup(dtype)
    oracle = OracleDecoder(cfg, w32)
    x, ids = reqs[0]
    first = eng.prefill(rb, [x], [ids])
    cache, lg = oracle.prefill(x, cap)
    st = SpecState(cache, x.shape[0], first[0], [first[0]], x.shape[0])
    assert float(lg.max() - lg[first[0]]) <= REL[dtype] * float(lg.abs().max())
    for _ in range(4):
        before = st.seq_len
        eng.round_launch(rb)
        torch.cuda.synchronize()
        eng.check_status(rb)
        am, v = rb.am.cpu(), rb.v.cpu()
        _rows_close(am, rb.top_d.cpu(), spec_draft(oracle, st, K)[1], REL[dtype])
        _rows_close(v, rb.top_v.cpu(), spec_verify(oracle, st, am.long())[1], REL[dtype])
        res = spec_commit(st, am.tolist(), v.tolist())
        pk = rb.packed.cpu()[0].tolist()
        assert pk[0] == int(am[0]) and pk[1] == res["acc"] and pk[2: 3 + pk[1]] == v[: pk[1] + 1].tolist()
        assert int(rb.seq_lens[0]) == st.seq_len == before + pk[1] + 2


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
def test_cache_holds_the_rows_the_attention_reads(dtype):
    """After a prefill the cache's rows, read back, are the quantised rotation of the engine's own last projection."""
    fmt = "int8" if dtype == torch.int8 else "e4m3"
    cfg, w32, reqs, eng, rb, cap = _setup(dtype, n_image=40, n_prompt=20)
    x, ids = reqs[0]
    eng.prefill(rb, [x], [ids])                     # one chunk of 64 rows: 60 and four padding ones
    torch.cuda.synchronize()
    n = x.shape[0]
    qkv = eng.qkv[:n].cpu().double().view(n, -1, 128)          # the last layer's
    ang = R.angles(eng.w.inv_freq.cpu(), torch.arange(n))
    k = R.norm_rotate(qkv[:, cfg.n_q_heads: cfg.n_q_heads + cfg.n_kv_heads], None, 0.0, ang, False)
    v = qkv[:, cfg.n_q_heads + cfg.n_kv_heads:]
    slots = rb.page_table[0].cpu().long()[torch.arange(n) // 16] * 16 + torch.arange(n) % 16
    out = torch.zeros((2, n, cfg.kv_dim), dtype=torch.bfloat16, device=DEV)
    L.kv_read(eng.kv[-1], slots.to(DEV), out[0], out[1])
    for o, ref in zip(out, (k, v)):
        assert torch.equal(o.double().cpu().view(n, -1, 128), R.values(*R.quantise(ref, fmt)))


@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn])
def test_graph_replay_equals_eager_and_batches_equal_single_requests(dtype):
    cfg, w32, reqs, eng, rb, cap = _setup(dtype, bs=3)
    eng.prefill(rb, [r[0] for r in reqs], [r[1] for r in reqs], attn_chunk=128)
    snap = (rb.seq_lens.clone(), rb.seeds.clone(), rb.n_committed.clone())
    eager = []
    for _ in range(3):
        eng.round_launch(rb)
        torch.cuda.synchronize()
        eager.append(rb.packed.cpu().clone())

    def rewind():
        for t, s in zip((rb.seq_lens, rb.seeds, rb.n_committed), snap):
            t.copy_(s)

    rewind()
    graph = eng.capture(rb)
    rewind()
    for want in eager:
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(rb.packed.cpu(), want)
    eng.check_status(rb)
    for b in range(3):
        _, _, _, one, rb1, _ = _setup(dtype, bs=1)
        one.prefill(rb1, [reqs[b][0]], [reqs[b][1]], attn_chunk=128)
        for want in eager:
            one.round_launch(rb1)
            torch.cuda.synchronize()
            assert rb1.packed.cpu()[0].tolist() == want[b].tolist()
        del one


def test_multimodal_positions_reach_the_write():
    """A prefix on an image grid: another rotation, another stream state; the engine runs it through row_pos3."""
    cfg, w32, reqs, eng, rb, cap = _setup(torch.int8)
    x, ids = reqs[0]
    pos3 = grid_positions(64, 16, 8)
    eng.prefill(rb, [x], [ids], prefix_pos3=[pos3])
    oracle = OracleDecoder(cfg, w32)
    cache, lg = oracle.prefill(x, cap, pos3)
    k = eng.pool.k[0].cpu().double() * 2.0 ** eng.pool.k_exp[0].cpu().double()[..., None]
    n = x.shape[0]
    slots = rb.page_table[0].cpu().long()[torch.arange(n) // 16] * 16 + torch.arange(n) % 16
    got = k.transpose(1, 2).flatten(0, 1)[slots]
    # layer 0's keys: bf16 projections (2^-8) of bf16-rounded inputs (2^-8), then half a code step (2^-8 of the row's largest)
    ref = cache.k[0, :n].double()
    assert ((got - ref).abs() <= 2.0 ** -8 * ref.abs().amax(-1, keepdim=True) * 4).all()


def test_memory_is_halved():
    cfg = small_model(2)
    assert PagePool.bytes_needed(cfg, 10, 16, torch.int8) * 256 == PagePool.bytes_needed(cfg, 10, 16) * 129
    with pytest.raises(ValueError, match="no K/V cache"):
        Engine(cfg, {}, max_rows=1, n_pages=1, kv_dtype=torch.float16)
