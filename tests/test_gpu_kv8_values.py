"""8-bit cache write and attention on values far from one: norms whose sums or products leave fp32, query rows of the largest and
smallest sizes; against the 64-bit oracle, codes equal, outputs within the bounds of test_gpu_kv8."""
import pytest
import torch

from gravityocr_b200 import _lib as L
from oracle import kv8_ref as R
from test_gpu_kv8 import DEV, _attend, _attn_case, _cache, _check_attention, _close_bf16, _rows, _status

pytestmark = pytest.mark.gpu

# (size of the rows, size of the weights, eps): squares, sums or products beyond fp32 or below its normal numbers
SIZES = [(1.0, 1.0, 1e-6), (2.0 ** 110, 2.0 ** 30, 1e-6), (2.0 ** 120, 2.0 ** -20, 1e-6), (2.0 ** 66, 1.0, 0.0),
         (2.0 ** 30, 2.0 ** 100, 1e-6), (2.0 ** -110, 2.0 ** -18, 0.0), (2.0 ** -70, 1.0, 0.0), (2.0 ** -70, 1.0, 1e-6),
         (2.0 ** -120, 2.0 ** 30, 0.0), (2.0 ** -40, 2.0 ** -20, 0.0), (2.0 ** 62, 2.0 ** 62, 1e-30)]


@pytest.mark.parametrize("fmt", ["bf16", "e4m3", "int8"])
@pytest.mark.parametrize("half,rd", [(False, 64), (True, 128), (False, 0)])
@pytest.mark.parametrize("size,weight,eps", SIZES)
def test_norms_of_any_size(fmt, half, rd, size, weight, eps):
    m, nq, nkv = 21, 5, 3
    g = torch.Generator().manual_seed(3)
    x = torch.randn((m, (nq + 2 * nkv) * 128), generator=g) * size
    x[3] = 0.0 if eps else x[3]                         # (0 / 0 otherwise)
    x[5, ::7] = torch.randn((x.shape[1] + 6) // 7, generator=g)    # two sizes in a row
    x = x.bfloat16()
    w = [((1 + 0.2 * torch.randn(128, generator=g)) * weight).bfloat16() for _ in range(2)]
    w[0][9], w[1][17] = 0.0, 0.0
    inv = (1.0 / 10000.0 ** (torch.arange(0, rd, 2, dtype=torch.float64) / max(rd, 1))).float()
    pos = torch.randint(0, 4096, (m,), generator=g, dtype=torch.int32)
    slots = torch.randperm(64, generator=g)[:m]
    cache, st = _cache(4, nkv, fmt), _status()
    q = torch.zeros((m, nq * 128), dtype=torch.bfloat16, device=DEV)
    L.qk_norm_rope_write(x.to(DEV), nq, L.kv_cache(*cache), slots.to(DEV), q, inv.to(DEV), rd, row_pos=pos.to(DEV),
                         rope_half=half, q_norm=w[0].to(DEV), k_norm=w[1].to(DEV), eps=eps, status=st)
    assert int(st) == 0
    y = x.double().view(m, -1, 128)
    ang = R.angles(inv, pos) if rd else None
    rq = R.norm_rotate(y[:, :nq], w[0], eps, ang, half)
    rk = R.norm_rotate(y[:, nq: nq + nkv], w[1], eps, ang, half)
    assert torch.isfinite(rq).all() and float(rq.abs().max()) < 1e38
    _close_bf16(q, rq)
    if fmt == "bf16":
        _close_bf16(_rows(cache[0], slots), rk)
    else:
        want, e = R.quantise(rk, fmt)
        assert torch.equal(_rows(cache[2], slots).long(), e)
        assert torch.equal(_rows(cache[0], slots).double(), want)


def _sized(fmt, K, size, back):
    """Query rows of size `size`, keys of size 2^back."""
    c = _attn_case(fmt, [300, 90], K, 4, 2, spread=0.0)
    ke = c["cache"][2]
    ke += back
    assert int(ke.min()) >= -40 and int(ke.max()) <= 40
    c["k"] = c["k"] * 2.0 ** back
    q = c["q"].float()
    c["q"] = (q / q.abs().max() * (1.9 * size)).bfloat16()
    return c


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("K", [1, 9])
@pytest.mark.parametrize("size", [2.0 ** -30, 2.0 ** -60, 2.0 ** -110, 2.0 ** -126])
def test_attention_of_small_query_rows(fmt, K, size):
    c = _sized(fmt, K, size, 33)
    _check_attention(c, _attend(c))


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("K", [1, 9])
@pytest.mark.parametrize("size", [2.0 ** n for n in (48, 52, 54, 56, 57, 58, 59, 60, 64, 80)])
def test_attention_of_large_query_rows(fmt, K, size):
    """Scores from 10^4 up, where a score's fp32 step passes one, then the weights' whole range: they are finite in fp32, and a row
    attends to its largest alone (where that is larger by 2^-8 of it, far more than any rounding)."""
    c = _sized(fmt, K, size, -33)
    out = _attend(c).double().cpu().view(2, K, 4, 128)
    for b in range(2):
        q = c["q"][b * K: (b + 1) * K].double().view(K, 4, 128)
        k, v = c["k"][c["slots"][b]], c["v"][c["slots"][b]]
        s = torch.einsum("jhd,thd->jht", q, k.repeat_interleave(2, 1)) / 128 ** 0.5
        lim = torch.tensor(R.row_limits(0, c["lens"][b], K))
        s[(torch.arange(k.shape[0])[None] >= lim[:, None])[:, None].expand(s.shape)] = -float("inf")
        top = torch.topk(s, 2, -1)
        sure = top.values[..., 0] - top.values[..., 1] > 2.0 ** -8 * top.values[..., 0].abs()
        assert sure.float().mean() > 0.5                  # of the inputs
        want = v.repeat_interleave(2, 1).transpose(0, 1)[torch.arange(4)[None], top.indices[..., 0]]
        err = (out[b] - want).abs()[sure]
        assert (err <= 2.0 ** -8 * want.abs()[sure] + 2.0 ** -14 * want.abs().amax(-1, keepdim=True).expand(want.shape)[sure]).all()


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("K", [1, 9])
@pytest.mark.parametrize("size", [2.0 ** 100, 2.0 ** 107, 2.0 ** 110, 2.0 ** 125, 2.0 ** 126, 2.0 ** 127])
def test_attention_of_the_largest_query_rows(fmt, K, size):
    """Up to bf16's largest number."""
    test_attention_of_large_query_rows(fmt, K, size)


@pytest.mark.parametrize("fmt", ["bf16", "int8"])
def test_an_odd_head_changes_no_other(fmt):
    """Rows with one head whose norm leaves fp32: its neighbours' outputs are those of the row without it, whether a warp or many
    share the row."""
    nq, nkv, m = 16, 8, 2600
    g = torch.Generator().manual_seed(8)
    x = torch.randn((m, (nq + 2 * nkv) * 128), generator=g).bfloat16()
    y = x.clone().view(m, -1, 128)
    for h in (2, nq + 1):
        y[:, h] *= 2.0 ** 80
    w = [(1 + 0.2 * torch.randn(128, generator=g)).bfloat16().to(DEV) for _ in range(2)]
    inv = (1.0 / 10000.0 ** (torch.arange(0, 64, 2, dtype=torch.float64) / 64)).float().to(DEV)
    pos = torch.randint(0, 4096, (m,), generator=g, dtype=torch.int32).to(DEV)

    def run(rows, lo, hi):
        n = hi - lo
        cache = _cache(n // 16 + 1, nkv, fmt)
        q = torch.zeros((n, nq * 128), dtype=torch.bfloat16, device=DEV)
        L.qk_norm_rope_write(rows.view(m, -1)[lo:hi].to(DEV), nq, L.kv_cache(*cache), torch.arange(n, device=DEV), q, inv, 64,
                             row_pos=pos[lo:hi], q_norm=w[0], k_norm=w[1], eps=1e-6)
        return [q.cpu().view(n, nq, 128)] + [_rows(t, torch.arange(n)) for t in cache if t is not None]

    plain, loud = run(x, 0, m), run(y, 0, m)
    others = [h for h in range(nq) if h != 2]
    assert torch.equal(plain[0][:, others], loud[0][:, others])
    others = [h for h in range(nkv) if h != 1]
    for a, b in zip(plain[1:], loud[1:]):
        assert torch.equal(a[:, others], b[:, others])
    for lo, hi in ((0, 1), (7, 20)):
        for a, b in zip(loud, run(y, lo, hi)):
            assert torch.equal(a[lo:hi], b)
