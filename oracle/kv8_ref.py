"""64-bit restatement of the 8-bit K/V cache path and of the token log probabilities (torch float64, CPU).

Cache row: 128 values, codes on the format's grid and one exponent e in [-40, 40], the smallest with
max|x| <= top * 2^e; a row with a NaN or an infinity has e = -128 and reads back as NaN.
"""
from __future__ import annotations

import math
from typing import Optional, Sequence, Tuple

import torch

TOP = {"e4m3": 448.0, "int8": 127.0}
BAD = -128


def grid(fmt: str) -> torch.Tensor:
    """Non-negative values of the codes, ascending; the index's parity is the code's."""
    if fmt == "int8":
        return torch.arange(128, dtype=torch.float64)
    v = [m / 512 for m in range(8)] + [(8 + m) / 8 * 2.0 ** (k - 7) for k in range(1, 16) for m in range(8)]
    return torch.tensor(v[:127], dtype=torch.float64)


def nearest(y: torch.Tensor, fmt: str) -> torch.Tensor:
    """y rounded to the grid, ties to the even code, saturated."""
    g = grid(fmt)
    a = y.abs().clamp_max(float(g[-1]))
    hi = torch.searchsorted(g, a.contiguous()).clamp_max(g.numel() - 1)
    lo = (hi - 1).clamp_min(0)
    dh, dl = g[hi] - a, a - g[lo]
    pick = torch.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    return torch.copysign(g[pick], y)


def quantise(x: torch.Tensor, fmt: str) -> Tuple[torch.Tensor, torch.Tensor]:
    """x [..., 128] float64 -> code values (float64), exponents (int64)."""
    bad = ~torch.isfinite(x).all(-1)
    x = torch.where(bad[..., None], torch.zeros_like(x), x)
    amax = x.abs().amax(-1)
    borders = torch.tensor([TOP[fmt] * 2.0 ** e for e in range(-40, 40)], dtype=torch.float64)
    e = -40 + torch.searchsorted(borders, amax.contiguous())
    codes = nearest(x / (2.0 ** e.double())[..., None], fmt)
    return codes, torch.where(bad, torch.full_like(e, BAD), e)


def values(codes: torch.Tensor, exps: torch.Tensor) -> torch.Tensor:
    e = exps.to(torch.int64)
    f = torch.where(e == BAD, torch.full(e.shape, float("nan"), dtype=torch.float64), 2.0 ** e.double())
    return codes.double() * f[..., None]


def angles(inv_freq: torch.Tensor, pos: Optional[torch.Tensor] = None, pos3: Optional[torch.Tensor] = None,
           section: Optional[Sequence[int]] = None) -> torch.Tensor:
    f = inv_freq.double()
    if pos3 is None:
        return pos.double()[:, None] * f
    axis = torch.tensor([a for a, n in enumerate(section) for _ in range(n)])
    return pos3.double()[:, axis] * f


def norm_rotate(x: torch.Tensor, w: Optional[torch.Tensor], eps: float, ang: Optional[torch.Tensor],
                half: bool) -> torch.Tensor:
    """x [m, heads, 128] float64: RMS norm (w given), then the rotation of the first 2 * ang.shape[1] elements."""
    y = x.clone()
    if w is not None:
        y = y / torch.sqrt((y * y).mean(-1, keepdim=True) + eps) * w.double()
    if ang is None or ang.shape[1] == 0:
        return y
    p = ang.shape[1]
    c, s = torch.cos(ang)[:, None], torch.sin(ang)[:, None]
    i0, i1 = (slice(0, p), slice(p, 2 * p)) if half else (slice(0, 2 * p, 2), slice(1, 2 * p, 2))
    a, b = y[..., i0].clone(), y[..., i1].clone()
    y[..., i0], y[..., i1] = a * c - b * s, b * c + a * s
    return y


def row_limits(draft: int, base: int, K: int):
    """Cache positions [0, limit) each window row sees."""
    if draft == 0:
        return [base + j + 1 for j in range(K)]
    return [base + 1 if (j == 0 and draft == 1) else base + K for j in range(K)]


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, base: int, draft: int) -> torch.Tensor:
    """q [K, n_q, 128], k / v [tokens, n_kv, 128] float64 -> [K, n_q, 128]; a row that sees nothing is zero."""
    K, nq, D = q.shape
    G = nq // k.shape[1]
    out = torch.zeros((K, nq, D), dtype=torch.float64)
    for j, lim in enumerate(row_limits(draft, base, K)):
        if lim <= 0:
            continue
        kk, vv = (t[:lim].repeat_interleave(G, dim=1) for t in (k, v))
        p = torch.softmax(torch.einsum("hd,thd->ht", q[j], kk) / math.sqrt(D), -1)
        out[j] = torch.einsum("ht,thd->hd", p, vv)
    return out


def logprobs(logits: torch.Tensor, ids: torch.Tensor, temperature: Optional[torch.Tensor], n_top: int):
    """(logprob, entropy, rank, top_logprob, top_ids) of rows that have a distribution; float64.  The best token's own 1
    stays out of the sum: next to it 64 bits would lose terms below 2^-53, and log1p does not need it."""
    x = logits.double()
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    d = x - x.gather(1, order[:, :1])
    if temperature is not None:
        d = d / temperature.double()[:, None]
    rest = d.exp().scatter(1, order[:, :1], 0.0)
    total = rest.sum(1)
    lp = d - torch.log1p(total)[:, None]
    ent = torch.log1p(total) - (rest * torch.where(rest > 0, d, torch.zeros_like(d))).sum(1) / (1 + total)
    rank = (order == ids[:, None]).long().argmax(1) + 1
    top = order[:, :n_top]
    return lp.gather(1, ids[:, None])[:, 0], ent, rank, lp.gather(1, top), top
