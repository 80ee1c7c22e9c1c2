"""Scratch buffers that captured graphs point to: they outlive the engine's growth, and nothing grows under a capture.
The engine is a shell without a GPU here (its launches are left out); tests/test_gpu_graph_scratch.py replays real graphs."""
import gc
import weakref

import pytest
import torch

from gravityocr_b200 import _lib as L
from gravityocr_b200.config import small_model
from gravityocr_b200.engine import Engine


@pytest.fixture
def shell(monkeypatch):
    """forward(capturing, bs, K, splits) of an engine on the CPU: sizes its scratch and keeps what it must."""
    state = {"capturing": False, "ws": None}
    monkeypatch.setattr(L, "embed_rows", lambda *a, **k: None)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state["capturing"])
    monkeypatch.setattr(Engine, "_forward_body", lambda self, *a: state.update(ws=a[-3]))

    def make(kv8):
        eng = object.__new__(Engine)
        eng.cfg, eng.kv8, eng.device, eng.max_rows, eng.page_size = small_model(2), kv8, torch.device("cpu"), 4096, 16
        eng.attn_ws = None
        eng._captured_scratch = []
        eng.lin_ws = torch.zeros((1,), dtype=torch.uint8)
        eng.y = torch.zeros((0,))
        z = torch.zeros((1,), dtype=torch.int32)
        eng.status = eng.x = eng.row_pos = eng.row_slot = eng.row_ids = z
        eng.h = [z, z]

        class W:
            embed, layers, inv_freq = z, [{"in": z}], z
        eng.w = W()

        def forward(capturing, bs, K, splits):
            state["capturing"] = capturing
            try:
                eng.forward(L.ROWS_EXPLICIT, bs, K, z, z, out_idx=z, attn_chunk=256, attn_splits=splits)
            finally:
                state["capturing"] = False
        return eng, forward, state
    return make


@pytest.mark.parametrize("kv8", [False, True])
def test_captured_scratch_outlives_growth(shell, kv8):
    eng, forward, state = shell(kv8)
    forward(False, 1, 17, 8)
    forward(True, 1, 17, 8)
    held = [weakref.ref(t) for t in (eng.attn_ws, eng.lin_ws, eng.y)]
    sizes = [t.numel() for t in (eng.attn_ws, eng.lin_ws, eng.y)]
    state["ws"] = None
    forward(False, 32, 64, 16)
    gc.collect()
    assert all(t.numel() > n for t, n in zip((eng.attn_ws, eng.y), (sizes[0], sizes[2])))   # they did grow
    assert all(r() is not None and r().numel() == n for r, n in zip(held, sizes))
    # what no graph points to goes
    free = weakref.ref(eng.attn_ws)
    state["ws"] = None
    forward(False, 64, 64, 16)
    gc.collect()
    assert free() is None


@pytest.mark.parametrize("kv8", [False, True])
def test_nothing_grows_under_a_capture(shell, kv8):
    eng, forward, _ = shell(kv8)
    eng.reserve(64)
    with pytest.raises(RuntimeError, match="attention workspace too small"):
        forward(True, 1, 17, 8)
    forward(True, 1, 17, 1)          # one split needs none
    forward(False, 1, 17, 8)
    forward(True, 1, 17, 8)
    with pytest.raises(RuntimeError, match="too small"):
        forward(True, 32, 64, 16)


def test_a_round_s_scratch_is_sized_before_its_capture(shell):
    eng, forward, _ = shell(True)

    class Rb:
        bs, K, attn_splits = 4, 17, 8
    eng._reserve_round(Rb)
    forward(True, 4, 17, 8)
    Rb.attn_splits, ws = 1, eng.attn_ws
    eng._reserve_round(Rb)
    assert eng.attn_ws is ws
