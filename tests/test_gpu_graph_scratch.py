"""A captured round on a B200 keeps its scratch: a larger prefill and a larger batch grow the engine's workspaces, memory that
is free afterwards is taken and overwritten by others, and the first graph still replays the rounds that an eager engine
runs, and writes nowhere else."""
import pytest
import torch

from gravityocr_b200.config import small_model
from gravityocr_b200.engine import Engine
from gravityocr_b200.weights import prefix_embeddings, random_weights, request_inputs

pytestmark = pytest.mark.gpu
DEV = "cuda"
K = 17


def _buffers(eng, bs, pages, attn_chunk):
    cap = pages * 16
    rb = eng.new_round_buffers(bs, K, pages, max_len=cap, avg_len=cap)
    rb.attn_chunk, rb.attn_splits = attn_chunk, -(-(cap + K + 1) // attn_chunk)
    for b in range(bs):
        rb.page_table[b] = torch.tensor(eng.pool.alloc(pages), dtype=torch.int32, device=DEV)
    return rb


@pytest.mark.parametrize("split_graphs", [False, True])
@pytest.mark.parametrize("dtype", [torch.int8, torch.float8_e4m3fn, torch.bfloat16])
def test_a_captured_round_survives_growth(dtype, split_graphs):
    cfg = small_model(2)
    w = random_weights(cfg, 0, torch.bfloat16)
    w32 = {k: v.float() for k, v in w.items()}
    reqs = []
    for b in range(6):
        img, txt = request_inputs(cfg, 0, 200, 24, b, torch.bfloat16)
        reqs.append((prefix_embeddings(w32, cfg, img, txt), torch.cat([torch.full((200,), -1, dtype=torch.int64), txt])))
    eng = Engine(cfg, w, max_rows=6 * 64, n_pages=200, kv_dtype=dtype)
    one = _buffers(eng, 1, 26, 128)
    eng.prefill(one, [reqs[0][0]], [reqs[0][1]], attn_chunk=128)
    state = (one.seq_lens, one.seeds, one.n_committed, one.rounds)
    snap = [t.clone() for t in state]

    def rewind():
        for t, s in zip(state, snap):
            t.copy_(s)

    want = []
    for _ in range(4):
        eng.round_launch(one)
        torch.cuda.synchronize()
        want.append(one.packed.cpu().clone())
    rewind()
    graphs = eng.capture_split(one) if split_graphs else (eng.capture(one),)
    before = eng.attn_ws.numel()
    many = _buffers(eng, 6, 26, 64)
    eng.prefill(many, [r[0] for r in reqs], [r[1] for r in reqs], attn_chunk=64)
    eng.round_launch(many)
    torch.cuda.synchronize()
    assert eng.attn_ws.numel() > before
    # whatever is free in the allocator's blocks, now with another owner
    free = torch.cuda.memory_reserved() - torch.cuda.memory_allocated()
    other, size = [], 1 << 25
    while size >= 512 and free > 0:
        if size > free:
            size >>= 1
            continue
        other.append(torch.full((size,), 0xA5, dtype=torch.uint8, device=DEV))
        free = min(free - size, torch.cuda.memory_reserved() - torch.cuda.memory_allocated())
    rewind()
    for row in want:
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(one.packed.cpu(), row)
    eng.check_status(one)
    assert all(bool((t == 0xA5).all()) for t in other)


def test_a_capture_that_would_grow_the_workspace_is_refused():
    cfg = small_model(2)
    eng = Engine(cfg, random_weights(cfg, 0, torch.bfloat16), max_rows=64, n_pages=64, kv_dtype=torch.int8)
    rb = _buffers(eng, 1, 26, 128)
    eng.reserve(K)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="attention workspace too small"):
        with torch.cuda.graph(graph):
            eng.verify_launch(rb)
    torch.cuda.synchronize()
    eng.capture(rb)          # sizes it first
    assert eng.attn_ws is not None
