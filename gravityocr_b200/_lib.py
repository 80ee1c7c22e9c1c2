"""ctypes binding of ``libgravity_b200.so`` (C ABI in ``include/gravity_b200.h``).

The wrappers take torch tensors, check dtype / device / contiguity, pass raw device pointers and the current CUDA
stream, and raise ``RuntimeError`` on any non-zero status.  There is no fallback: if the library is missing or
fails to load, every call raises.
"""
from __future__ import annotations

import ctypes
import os
import threading
from typing import Optional

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.environ.get("GRAVITY_B200_LIB", os.path.join(_HERE, "libgravity_b200.so"))

GR_OK = 0
EPI_STORE_F32, EPI_STORE_BF16, EPI_SWIGLU, EPI_QKV_ROPE, EPI_ARGMAX, EPI_PARTIAL_F32 = range(6)
ROWS_DRAFT, ROWS_VERIFY, ROWS_EXPLICIT = range(3)

# every symbol include/gravity_b200.h declares
EXPORTS = ("gr_version", "gr_status_string", "gr_set_pdl", "gr_set_attention_tc", "gr_num_sms", "gr_linear_workspace_bytes",
           "gr_attention_workspace_bytes", "gr_linear_default_splits", "gr_linear_plan", "gr_linear", "gr_embed_rows",
           "gr_residual_norm", "gr_bd_attention", "gr_accept_commit", "gr_draft_override", "gr_pack_gate_up",
           "gr_bd_attention_noalloc", "gr_bd_attention_ordered", "gr_gather_rows", "gr_logits_process",
           "gr_sample_rows", "gr_commit_sampled", "gr_penalty_cumulate", "gr_qk_norm_rope_write", "gr_kv_read",
           "gr_kv8_attention_workspace_bytes", "gr_kv8_attention_plan", "gr_kv8_attention", "gr_token_logprobs")
FILTER_JOINT, FILTER_SEQUENTIAL, FILTER_TORCH = range(3)
PEN_REPETITION, PEN_FREQUENCY, PEN_PRESENCE, PEN_MIN_NEW_TOKENS = range(4)
COIN_ACCEPT, COIN_FINAL, COIN_FIRST, COIN_PREFILL = range(4)
GR_ERR_NO_TOKEN = 9


class Epilogue(ctypes.Structure):
    _fields_ = [
        ("mode", ctypes.c_int),
        ("out", ctypes.c_void_p),
        ("ld_out", ctypes.c_int),
        ("q_out", ctypes.c_void_p),
        ("k_cache", ctypes.c_void_p),
        ("v_cache", ctypes.c_void_p),
        ("row_pos", ctypes.c_void_p),
        ("row_slot", ctypes.c_void_p),
        ("inv_freq", ctypes.c_void_p),
        ("rotary_dim", ctypes.c_int),
        ("n_q_heads", ctypes.c_int),
        ("n_kv_heads", ctypes.c_int),
        ("page_size", ctypes.c_int),
        ("out_idx", ctypes.c_void_p),
        ("out_top1", ctypes.c_void_p),
        ("out_gap", ctypes.c_void_p),
        ("row_pos3", ctypes.c_void_p),
        ("mrope_section", ctypes.c_int * 3),
    ]


class Sampling(ctypes.Structure):
    """gr_sampling: per-request parameter arrays, penalizer state by pool slot, grammar mask, bias and the coins' rng."""
    _fields_ = [
        ("vocab", ctypes.c_int),
        ("filter", ctypes.c_int),
        ("temperature", ctypes.c_void_p),
        ("top_k", ctypes.c_void_p),
        ("top_p", ctypes.c_void_p),
        ("min_p", ctypes.c_void_p),
        ("n_order", ctypes.c_int),
        ("order", ctypes.c_int * 4),
        ("repetition", ctypes.c_void_p),
        ("frequency", ctypes.c_void_p),
        ("presence", ctypes.c_void_p),
        ("min_new_tokens", ctypes.c_void_p),
        ("stop_ids", ctypes.c_void_p),
        ("n_stop", ctypes.c_int),
        ("st_rep", ctypes.c_void_p),
        ("st_freq", ctypes.c_void_p),
        ("st_pres", ctypes.c_void_p),
        ("st_len", ctypes.c_void_p),
        ("req_pool_idx", ctypes.c_void_p),
        ("allowed", ctypes.c_void_p),
        ("logit_bias", ctypes.c_void_p),
        ("rng", ctypes.c_void_p),
    ]


class KvCache(ctypes.Structure):
    """gr_kv_cache: one layer's paged K/V cache in bf16, e4m3 or int8 (made by ``kv_cache``)."""
    _fields_ = [
        ("format", ctypes.c_int),
        ("n_kv_heads", ctypes.c_int),
        ("page_size", ctypes.c_int),
        ("n_pages", ctypes.c_int64),
        ("k", ctypes.c_void_p),
        ("v", ctypes.c_void_p),
        ("k_exp", ctypes.c_void_p),
        ("v_exp", ctypes.c_void_p),
    ]


_lib = None
_lock = threading.Lock()

_P, _I, _Z, _F, _L = ctypes.c_void_p, ctypes.c_int, ctypes.c_size_t, ctypes.c_float, ctypes.c_int64
_SIGS = {
    "gr_version": (_I, []),
    "gr_status_string": (ctypes.c_char_p, [_I]),
    "gr_set_pdl": (None, [_I]),
    "gr_set_attention_tc": (None, [_I]),
    "gr_num_sms": (_I, []),
    "gr_linear_workspace_bytes": (_Z, [_I, _I, _I]),
    "gr_attention_workspace_bytes": (_Z, [_I, _I, _I, _I, _I]),
    "gr_linear_default_splits": (_I, [_I, _I, _I, _I]),
    "gr_linear_plan": (_I, [_I, _I, _I, _I, _I, _P]),
    "gr_linear": (_I, [_P, _I, _I, _P, _I, ctypes.POINTER(Epilogue), _I, _P, _Z, _P, _Z, _P, _P]),
    "gr_embed_rows": (_I, [_I, _I, _I, _P, _P, _P, _P, _P, _P, _P, _I, _I, _I, _P, _I, _I, _P, _F, _I, _P, _P, _P,
                           _P, _P, _P, _P, _P]),
    "gr_residual_norm": (_I, [_I, _I, _P, _P, _I, _P, _P, _F, _P, _P, _P]),
    "gr_bd_attention": (_I, [_P, _P, _P, _L, _P, _I, _P, _I, _I, _I, _I, _I, _I, _I, _I, _I, _P, _P, _Z, _P, _P]),
    "gr_accept_commit": (_I, [_I, _I, _P, _P, _P, _P, _P, _I, _P, _P, _P, _P, _P, _P, _P, _P, _P]),
    "gr_draft_override": (_I, [_I, _I, _P, _P, _I, _P, _P, _I, _P, _I, _I, _P]),
    "gr_pack_gate_up": (_I, [_P, _P, _I, _I, _P]),
    "gr_bd_attention_noalloc": (_I, [_P, _P, _P, _L, _P, _I, _P, _I, _I, _I, _I, _I, _I, _I, _I, _I, _P, _P, _P]),
    "gr_gather_rows": (_I, [_P, _I, _I, _I, _P, _P]),
    "gr_logits_process": (_I, [_P, _I, _I, _P, ctypes.POINTER(Sampling), _P]),
    "gr_sample_rows": (_I, [_P, _I, _I, _P, ctypes.POINTER(Sampling), _I, _P, _P, _P, _P, _I, _P, _P]),
    "gr_commit_sampled": (_I, [_I, _I, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P]),
    "gr_penalty_cumulate": (_I, [_I, _P, _I, _P, _I, ctypes.POINTER(Sampling), _P]),
    "gr_bd_attention_ordered": (_I, [_P, _P, _P, _L, _P, _I, _P, _P, _I, _I, _I, _I, _I, _I, _I, _I, _I, _P, _P, _Z, _P,
                                     _P]),
    "gr_qk_norm_rope_write": (_I, [_P, _L, _I, _I, ctypes.POINTER(KvCache), _P, _P, ctypes.c_double, _P, _P, _P, _P, _I, _I,
                                   _P, _P, _P, _P]),
    "gr_kv_read": (_I, [ctypes.POINTER(KvCache), _P, _L, _P, _P, _P, _P]),
    "gr_kv8_attention_workspace_bytes": (_Z, [_I, _I, _I, _I, _I]),
    "gr_kv8_attention_plan": (_I, [_I, _I, _I, _I, _I, _P]),
    "gr_kv8_attention": (_I, [_P, ctypes.POINTER(KvCache), _P, _I, _P, _I, _I, _I, _I, _I, _I, _I, _P, _P, _Z, _P, _P]),
    "gr_token_logprobs": (_I, [_P, _I, _L, _I, _I, _P, _P, _I, _P, _P, _P, _P, _P, _P, _P]),
}
GR_ERR_SCRATCH_LIMIT = 8
NOALLOC_SCRATCH_BYTES = 8 << 20


def load(path: Optional[str] = None):
    """Load the library (once).  Raises if it is missing: there is no CPU or library fallback."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is not None:
            return _lib
        p = path or LIB_PATH
        if not os.path.exists(p):
            raise RuntimeError(f"libgravity_b200.so not found at {p}: build it with `python -m gravityocr_b200.build`")
        lib = ctypes.CDLL(p)
        for name, (res, args) in _SIGS.items():
            f = getattr(lib, name)
            f.restype = res
            f.argtypes = args
        _lib = lib
        return lib


def _check(rc: int, what: str) -> None:
    if rc != GR_OK:
        raise RuntimeError(f"{what} failed: {load().gr_status_string(rc).decode()} (code {rc})")


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _stream(stream=None) -> int:
    s = stream if stream is not None else torch.cuda.current_stream()
    return s.cuda_stream


def _need(t: torch.Tensor, dtype: torch.dtype, name: str) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    if t.dtype != dtype:
        raise RuntimeError(f"{name} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous")


# ---------------------------------------------------------------------- wrappers
def set_pdl(enable: bool) -> None:
    load().gr_set_pdl(1 if enable else 0)


def set_attention_tc(mode) -> None:
    """Attention kernel: 0 / False mma.sync everywhere; 1 / True tcgen05 on grids of more than one CTA per SM (the
    default); 2 tcgen05 on every grid."""
    load().gr_set_attention_tc(int(mode))


def num_sms() -> int:
    return int(load().gr_num_sms())


def linear_workspace_bytes(n_out: int, m: int, splits: int) -> int:
    return int(load().gr_linear_workspace_bytes(n_out, m, splits))


def linear_default_splits(n_out: int, k_in: int, m: int, mode: int = EPI_STORE_F32) -> int:
    """Split-K count gr_linear plans for this shape and epilogue mode."""
    return int(load().gr_linear_default_splits(n_out, k_in, m, mode))


def linear_plan(n_out: int, k_in: int, m: int, mode: int = EPI_STORE_F32, splits: int = 0) -> dict:
    """The plan gr_linear runs for this call: split count, token-tile height and count, unit order, grid."""
    out = (ctypes.c_int32 * 5)()
    _check(load().gr_linear_plan(n_out, k_in, m, mode, splits, out), "gr_linear_plan")
    return {"splits": out[0], "nt": out[1], "m_tiles": out[2], "tail_last": bool(out[3]), "grid": out[4]}


def attention_workspace_bytes(bs: int, K: int, n_q_heads: int, n_kv_heads: int, max_splits: int) -> int:
    return int(load().gr_attention_workspace_bytes(bs, K, n_q_heads, n_kv_heads, max_splits))


def linear(w: torch.Tensor, x: torch.Tensor, m: int, epi: Epilogue, workspace: torch.Tensor, splits: int = 0,
           prefetch: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None, stream=None) -> None:
    _need(w, torch.bfloat16, "w")
    _need(x, torch.bfloat16, "x")
    n_out, k_in = w.shape
    if x.shape[-1] != k_in or x.numel() < m * k_in:
        raise RuntimeError(f"x shape {tuple(x.shape)} does not match w {tuple(w.shape)} with m={m}")
    rc = load().gr_linear(w.data_ptr(), n_out, k_in, x.data_ptr(), m, ctypes.byref(epi), splits,
                          workspace.data_ptr(), workspace.numel() * workspace.element_size(),
                          _ptr(prefetch), 0 if prefetch is None else prefetch.numel() * prefetch.element_size(),
                          _ptr(status), _stream(stream))
    _check(rc, "gr_linear")


def embed_rows(mode: int, bs: int, K: int, *, seeds=None, rpi=None, ids32=None, ids64=None, row_embeds=None,
               seq_lens, page_table, page_size: int, embed, vocab: int, mask_id: int, norm_w, eps: float,
               h_out, x_out, row_pos, row_slot, row_ids=None, rope_delta=None, status=None, stream=None) -> None:
    rc = load().gr_embed_rows(mode, bs, K, _ptr(seeds), _ptr(rpi), _ptr(ids32), _ptr(ids64), _ptr(row_embeds),
                              seq_lens.data_ptr(), page_table.data_ptr(), page_table.shape[1], page_size,
                              page_table.shape[1], embed.data_ptr(), vocab, mask_id, norm_w.data_ptr(), eps,
                              embed.shape[1], h_out.data_ptr(), x_out.data_ptr(), row_pos.data_ptr(),
                              row_slot.data_ptr(), _ptr(row_ids), _ptr(rope_delta), _ptr(status), _stream(stream))
    _check(rc, "gr_embed_rows")


def residual_norm(m: int, h_in, y, w_a, w_b, eps: float, h_out, x_out, y_parts: int = 1, stream=None) -> None:
    rc = load().gr_residual_norm(m, h_in.shape[-1], h_in.data_ptr(), y.data_ptr(), y_parts, w_a.data_ptr(),
                                 w_b.data_ptr(), eps, h_out.data_ptr(), x_out.data_ptr(), _stream(stream))
    _check(rc, "gr_residual_norm")


def bd_attention(q, k_cache, v_cache, page_table, seq_lens, bs: int, K: int, draft, base_add: int,
                 n_q_heads: int, n_kv_heads: int, page_size: int, chunk: int, max_splits: int, out, workspace,
                 status=None, stream=None, order=None) -> None:
    n_pages = k_cache.shape[0]
    rc = load().gr_bd_attention_ordered(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), n_pages,
                                page_table.data_ptr(), page_table.shape[1], seq_lens.data_ptr(), _ptr(order),
                                bs, K, int(draft), base_add,
                                n_q_heads, n_kv_heads, page_size, chunk, max_splits, out.data_ptr(),
                                _ptr(workspace), 0 if workspace is None else workspace.numel() * workspace.element_size(),
                                _ptr(status), _stream(stream))
    _check(rc, "gr_bd_attention")


def accept_commit(bs: int, K: int, am, v, seeds, rpi, seq_lens, packed, released, out_next, *, x0_committed=False,
                  loc=None, n_released=None, n_committed=None, rounds=None, accept_len=None, stream=None) -> None:
    rc = load().gr_accept_commit(bs, K, am.data_ptr(), v.data_ptr(), seeds.data_ptr(), rpi.data_ptr(),
                                 seq_lens.data_ptr(), 1 if x0_committed else 0, _ptr(loc), packed.data_ptr(),
                                 released.data_ptr(), _ptr(n_released), out_next.data_ptr(), _ptr(n_committed),
                                 _ptr(rounds), _ptr(accept_len), _stream(stream))
    _check(rc, "gr_accept_commit")


def draft_override(bs: int, K: int, am, g, n_committed, plan, rounds, vocab: int, mask_id: int, stream=None) -> None:
    rc = load().gr_draft_override(bs, K, am.data_ptr(), g.data_ptr(), g.shape[1], n_committed.data_ptr(),
                                  plan.data_ptr(), plan.shape[1], rounds.data_ptr(), vocab, mask_id, _stream(stream))
    _check(rc, "gr_draft_override")


def pack_gate_up(src: torch.Tensor, dst: torch.Tensor, intermediate: int, stream=None) -> None:
    _need(src, torch.bfloat16, "src")
    _need(dst, torch.bfloat16, "dst")
    rc = load().gr_pack_gate_up(src.data_ptr(), dst.data_ptr(), intermediate, src.shape[1], _stream(stream))
    _check(rc, "gr_pack_gate_up")


def bd_attention_noalloc(q, k_cache, v_cache, page_table, seq_lens, bs: int, K: int, draft, base_add: int,
                         n_q_heads: int, n_kv_heads: int, page_size: int, chunk: int, max_splits: int, out,
                         status=None, stream=None) -> None:
    """``bd_attention`` for callers that cannot allocate device memory: the split scratch is the library's own
    fixed 8 MiB device array (see ``gr_bd_attention_noalloc`` in include/gravity_b200.h for the limits)."""
    rc = load().gr_bd_attention_noalloc(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), k_cache.shape[0],
                                        page_table.data_ptr(), page_table.shape[1], seq_lens.data_ptr(), bs, K,
                                        int(draft), base_add, n_q_heads, n_kv_heads, page_size, chunk,
                                        max_splits, out.data_ptr(), _ptr(status), _stream(stream))
    _check(rc, "gr_bd_attention_noalloc")


# ---------------------------------------------------------------------- non-greedy rounds
def gather_rows(src: torch.Tensor, n: int, stride_rows: int, dst: torch.Tensor, stream=None) -> None:
    row_bytes = src.shape[-1] * src.element_size()
    _check(load().gr_gather_rows(src.data_ptr(), row_bytes, n, stride_rows, dst.data_ptr(), _stream(stream)),
           "gr_gather_rows")


def logits_process(logits: torch.Tensor, bs: int, K: int, cand, smp: Sampling, stream=None) -> None:
    _need(logits, torch.float32, "logits")
    _check(load().gr_logits_process(logits.data_ptr(), bs, K, _ptr(cand), ctypes.byref(smp), _stream(stream)),
           "gr_logits_process")


def sample_rows(logits: torch.Tensor, bs: int, K: int, cand, smp: Sampling, first_kind: int, accept, sample,
                p_next=None, first_out=None, first_stride: int = 1, status=None, stream=None) -> None:
    _need(logits, torch.float32, "logits")
    _check(load().gr_sample_rows(logits.data_ptr(), bs, K, _ptr(cand), ctypes.byref(smp), first_kind, _ptr(accept),
                                 sample.data_ptr(), _ptr(p_next), _ptr(first_out), first_stride, _ptr(status),
                                 _stream(stream)), "gr_sample_rows")


def commit_sampled(bs: int, K: int, am, accept, sample, seeds, rpi, seq_lens, predict, packed, released, out_next, *,
                   n_released=None, n_committed=None, rounds=None, accept_len=None, rng=None, stream=None) -> None:
    _check(load().gr_commit_sampled(bs, K, am.data_ptr(), accept.data_ptr(), sample.data_ptr(), seeds.data_ptr(),
                                    rpi.data_ptr(), seq_lens.data_ptr(), predict.data_ptr(), packed.data_ptr(),
                                    released.data_ptr(), _ptr(n_released), out_next.data_ptr(), _ptr(n_committed),
                                    _ptr(rounds), _ptr(accept_len), _ptr(rng), _stream(stream)), "gr_commit_sampled")


def penalty_cumulate(bs: int, tokens, stride: int, counts, add: int, smp: Sampling, stream=None) -> None:
    _check(load().gr_penalty_cumulate(bs, tokens.data_ptr(), stride, _ptr(counts), add, ctypes.byref(smp),
                                      _stream(stream)), "gr_penalty_cumulate")


# ---------------------------------------------------------------------- 8-bit K/V cache
KV_BF16, KV_E4M3, KV_INT8 = range(3)
_KV_FORMATS = {torch.bfloat16: KV_BF16, torch.float8_e4m3fn: KV_E4M3, torch.int8: KV_INT8}


def _bad(t: torch.Tensor, dtype: torch.dtype, device: int, n: int, name: str, exact: bool) -> None:
    """What is wrong with an argument that ``_arg`` did not take."""
    _need(t, dtype, name)
    if t.get_device() != device:
        raise RuntimeError(f"{name} is on cuda:{t.get_device()}, the call's other tensors on cuda:{device}")
    raise RuntimeError(f"{name} holds {t.numel()} elements, the call needs {'' if exact else 'at least '}{n}")


def _arg(t: torch.Tensor, dtype: torch.dtype, device: int, n: int, name: str) -> int:
    """Pointer of a contiguous tensor of n elements on the call's device."""
    if t.dtype is not dtype or t.get_device() != device or t.numel() != n or not t.is_contiguous():
        _bad(t, dtype, device, n, name, True)
    return t.data_ptr()


def _arg_least(t: torch.Tensor, dtype: torch.dtype, device: int, n: int, name: str) -> int:
    if t.dtype is not dtype or t.get_device() != device or t.numel() < n or not t.is_contiguous():
        _bad(t, dtype, device, n, name, False)
    return t.data_ptr()


def _call(device: int, stream, fn, *args) -> int:
    """fn(*args, stream) with ``device`` current, on the given stream or the device's current one."""
    if device == torch._C._cuda_getDevice():
        return fn(*args, torch._C._cuda_getCurrentRawStream(device) if stream is None else stream.cuda_stream)
    with torch.cuda.device(device):
        return fn(*args, _stream(stream))


def kv_cache(k: torch.Tensor, v: torch.Tensor, k_exp: Optional[torch.Tensor] = None,
             v_exp: Optional[torch.Tensor] = None) -> KvCache:
    """One layer's cache over the caller's tensors: k / v [pages, kv_heads, 16, 128] in bf16, float8_e4m3fn or int8 (the
    dtype is the format), and for the 8-bit formats k_exp / v_exp int8 [pages, kv_heads, 16].  The handle keeps the
    tensors alive."""
    if k.dtype not in _KV_FORMATS:
        raise RuntimeError(f"no cache format for {k.dtype}")
    _need(k, k.dtype, "k")
    _need(v, k.dtype, "v")
    if k.dim() != 4 or tuple(k.shape[2:]) != (16, 128) or v.shape != k.shape:
        raise RuntimeError(f"k / v must be [pages, kv_heads, 16, 128], got {tuple(k.shape)} / {tuple(v.shape)}")
    c = KvCache()
    c.format = _KV_FORMATS[k.dtype]
    if (c.format == KV_BF16) != (k_exp is None) or (k_exp is None) != (v_exp is None):
        raise RuntimeError("8-bit caches need k_exp and v_exp, a bf16 cache takes neither")
    for t, name in ((k_exp, "k_exp"), (v_exp, "v_exp")):
        if t is not None:
            _need(t, torch.int8, name)
            if t.shape != k.shape[:3]:
                raise RuntimeError(f"{name} must be {tuple(k.shape[:3])}, got {tuple(t.shape)}")
    for t, name in ((v, "v"), (k_exp, "k_exp"), (v_exp, "v_exp")):
        if t is not None and t.device != k.device:
            raise RuntimeError(f"{name} is on {t.device}, k on {k.device}")
    c.n_pages, c.n_kv_heads, c.page_size = k.shape[0], k.shape[1], 16
    c.k, c.v, c.k_exp, c.v_exp = _ptr(k), _ptr(v), _ptr(k_exp), _ptr(v_exp)
    c.tensors = (k, v, k_exp, v_exp)
    c.device = k.get_device()
    return c


def qk_norm_rope_write(qkv: torch.Tensor, n_q_heads: int, cache: KvCache, row_slot: torch.Tensor, q_out: torch.Tensor,
                       inv_freq: Optional[torch.Tensor], rotary_dim: int, *, row_pos=None, row_pos3=None,
                       mrope_section=None, rope_half: bool = False, q_norm=None, k_norm=None, eps: float = 1e-5,
                       status=None, stream=None) -> None:
    """Projected rows qkv [m, >= (n_q_heads + 2 kv_heads) * 128] bf16 (a row stride is allowed): per-head norms of q and k
    (optional), the rotation, q to q_out, k and v to the cache at row_slot (gr_qk_norm_rope_write)."""
    if qkv.dtype is not torch.bfloat16 or qkv.dim() != 2 or not qkv.is_cuda or (qkv.shape[1] > 1 and qkv.stride(1) != 1):
        raise RuntimeError("qkv must be a CUDA bf16 [m, width] tensor with unit column stride")
    dev = cache.device
    m, width = qkv.shape
    heads = n_q_heads + 2 * cache.n_kv_heads
    if m < 1 or n_q_heads < 1 or width < heads * 128:
        raise RuntimeError(f"qkv {tuple(qkv.shape)} does not hold {heads} heads of 128")
    if qkv.get_device() != dev:
        raise RuntimeError(f"qkv is on {qkv.device}, the cache on cuda:{dev}")
    rc = _call(dev, stream, load().gr_qk_norm_rope_write, qkv.data_ptr(), qkv.stride(0) if m > 1 else width, m, n_q_heads,
               ctypes.byref(cache),
               None if q_norm is None else _arg(q_norm, torch.bfloat16, dev, 128, "q_norm"),
               None if k_norm is None else _arg(k_norm, torch.bfloat16, dev, 128, "k_norm"), eps,
               None if row_pos is None else _arg(row_pos, torch.int32, dev, m, "row_pos"),
               None if row_pos3 is None else _arg(row_pos3, torch.int32, dev, 3 * m, "row_pos3"),
               None if mrope_section is None else (ctypes.c_int32 * 3)(*mrope_section),
               None if inv_freq is None else _arg(inv_freq, torch.float32, dev, rotary_dim // 2, "inv_freq"), rotary_dim,
               1 if rope_half else 0, _arg(row_slot, torch.int64, dev, m, "row_slot"),
               _arg(q_out, torch.bfloat16, dev, m * n_q_heads * 128, "q_out"),
               None if status is None else _arg_least(status, torch.int32, dev, 1, "status"))
    if rc:
        _check(rc, "gr_qk_norm_rope_write")


def kv_read(cache: KvCache, slots: torch.Tensor, k_out: torch.Tensor, v_out: torch.Tensor, *, status=None,
            stream=None) -> None:
    """Cache rows at ``slots`` (int64 [n]) back in bf16: k_out / v_out [n, kv_heads * 128] (gr_kv_read)."""
    dev, n = cache.device, slots.numel()
    out = n * cache.n_kv_heads * 128
    rc = _call(dev, stream, load().gr_kv_read, ctypes.byref(cache), _arg(slots, torch.int64, dev, n, "slots"), n,
               _arg(k_out, torch.bfloat16, dev, out, "k_out"), _arg(v_out, torch.bfloat16, dev, out, "v_out"),
               None if status is None else _arg_least(status, torch.int32, dev, 1, "status"))
    if rc:
        _check(rc, "gr_kv_read")


def kv8_attention_workspace_bytes(bs: int, K: int, n_q_heads: int, n_kv_heads: int, max_splits: int) -> int:
    return int(load().gr_kv8_attention_workspace_bytes(bs, K, n_q_heads, n_kv_heads, max_splits))


def kv8_attention_split(bs: int, K: int, max_len: int, n_q_heads: int, n_kv_heads: int):
    """(chunk, splits) of kv8_attention for requests of up to ``max_len`` tokens, the K new rows included."""
    out = (ctypes.c_int32 * 2)()
    _check(load().gr_kv8_attention_plan(bs, K, max_len, n_q_heads, n_kv_heads, out), "gr_kv8_attention_plan")
    return out[0], out[1]


def kv8_attention(q: torch.Tensor, cache: KvCache, page_table: torch.Tensor, seq_lens: torch.Tensor, bs: int, K: int,
                  draft: int, base_add: int, n_q_heads: int, chunk: int, max_splits: int, out: torch.Tensor,
                  workspace: Optional[torch.Tensor], *, status=None, stream=None) -> None:
    """``bd_attention`` over an 8-bit cache; K = 1 is the attention of one new token (gr_kv8_attention)."""
    dev, n = cache.device, bs * K * n_q_heads * 128
    if page_table.dim() != 2 or page_table.shape[0] < bs:
        raise RuntimeError(f"page_table {tuple(page_table.shape)} holds fewer than {bs} requests")
    pages = page_table.shape[1]
    if workspace is None:
        ws, ws_bytes = None, 0
    else:
        ws_bytes = workspace.numel() * workspace.element_size()
        ws = _arg_least(workspace, workspace.dtype, dev, 0, "workspace")
    rc = _call(dev, stream, load().gr_kv8_attention, _arg_least(q, torch.bfloat16, dev, n, "q"),
               ctypes.byref(cache),
               _arg_least(page_table, torch.int32, dev, bs * pages, "page_table"), pages,
               _arg_least(seq_lens, torch.int64, dev, bs, "seq_lens"), bs, K, int(draft), base_add, n_q_heads, chunk,
               max_splits, _arg_least(out, torch.bfloat16, dev, n, "out"), ws, ws_bytes,
               None if status is None else _arg_least(status, torch.int32, dev, 1, "status"))
    if rc:
        _check(rc, "gr_kv8_attention")


# ---------------------------------------------------------------------- log probabilities
def token_logprobs(logits: torch.Tensor, ids: torch.Tensor, logprob: torch.Tensor, entropy: torch.Tensor,
                   rank: torch.Tensor, *, top_logprob: Optional[torch.Tensor] = None,
                   top_ids: Optional[torch.Tensor] = None, temperature: Optional[torch.Tensor] = None, status=None,
                   stream=None) -> None:
    """Log probability, rank and entropy of ids [rows] under softmax(logits / temperature), and the best alternatives into
    top_logprob / top_ids [rows, n].  logits: fp32 or bf16 [rows, vocab]; a row stride is allowed (gr_token_logprobs)."""
    bf16 = logits.dtype is torch.bfloat16
    if not (bf16 or logits.dtype is torch.float32) or logits.dim() != 2 or not logits.is_cuda or (
            logits.shape[1] > 1 and logits.stride(1) != 1):
        raise RuntimeError("logits must be a CUDA fp32 or bf16 [rows, vocab] tensor with unit column stride")
    rows, vocab = logits.shape
    dev, n_top, top, tid = logits.get_device(), 0, None, None
    if (top_logprob is None) != (top_ids is None):
        raise RuntimeError("top_logprob and top_ids come together")
    if top_ids is not None:
        if top_ids.dim() != 2 or top_ids.shape[0] != rows or top_logprob.shape != top_ids.shape:
            raise RuntimeError(f"top_logprob / top_ids must be [{rows}, n]")
        n_top = top_ids.shape[1]
        top = _arg(top_logprob, torch.float32, dev, rows * n_top, "top_logprob")
        tid = _arg(top_ids, torch.int32, dev, rows * n_top, "top_ids")
    rc = _call(dev, stream, load().gr_token_logprobs, logits.data_ptr(), bf16, logits.stride(0) if rows > 1 else vocab, rows,
               vocab, _arg(ids, torch.int64, dev, rows, "ids"),
               None if temperature is None else _arg(temperature, torch.float32, dev, rows, "temperature"), n_top,
               _arg(logprob, torch.float32, dev, rows, "logprob"), _arg(entropy, torch.float32, dev, rows, "entropy"),
               _arg(rank, torch.int32, dev, rows, "rank"), top, tid,
               None if status is None else _arg_least(status, torch.int32, dev, 1, "status"))
    if rc:
        _check(rc, "gr_token_logprobs")
