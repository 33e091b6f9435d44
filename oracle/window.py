"""Sliding-window attention with sinks in 64 bits.

TEST INFRASTRUCTURE ONLY: the oracle of ``cast_window_attention`` and
``cast_paged_window_attention``; nothing in the product imports it.
"""

from __future__ import annotations

import math

import torch


def sees(length: int, lq: int, window, sinks: int, frame: int, device=None) -> torch.Tensor:
    """bool ``[lq, length]``: key j is visible to query i at position
    ``length - lq + i``."""
    p = torch.arange(length - lq, length, device=device).unsqueeze(1)
    j = torch.arange(length, device=device).unsqueeze(0)
    fp, fj = torch.div(p, frame, rounding_mode="floor"), j // frame
    near = torch.ones_like(fj > fp) if window is None else (fp - fj < window)
    return (p >= 0) & (fj <= fp) & (near | (fj < sinks))


def attention(q, k, v, seen, scale=None):
    """One head: q ``[lq,D]``, k, v ``[n,D]``, seen ``[lq,n]`` -> float64
    ``(out, sum_j p_j |v_j|, largest |score|, largest sum_d |q_d k_d| scale)``,
    the last two ``[lq,1]``.  Rows and values that are not seen never enter;
    a row that sees nothing is zeros."""
    q, k, v = (t.to(torch.float64) for t in (q, k, v))
    scale = 1.0 / math.sqrt(q.shape[-1]) if scale is None else scale
    used = seen.any(0)
    k, v, seen = k[used], v[used], seen[:, used]
    s = (q @ k.mT * scale).masked_fill(~seen, -math.inf)
    m = s.amax(-1, keepdim=True) if s.shape[1] else torch.full((len(q), 1), -math.inf, dtype=s.dtype, device=s.device)
    e = torch.where(seen, torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m)), torch.zeros_like(s))
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total == 0, torch.ones_like(total), total)
    # a value that a row does not see has no weight at all, infinities included
    finite = torch.isfinite(v)
    out = p @ torch.where(finite, v, torch.zeros_like(v))
    size = p @ torch.where(finite, v, torch.zeros_like(v)).abs()
    for j in torch.nonzero(~finite.all(-1)).flatten().tolist():
        bad = torch.where(finite[j], torch.zeros_like(v[j]), v[j])
        out = out + torch.where(seen[:, j:j + 1], bad, torch.zeros_like(bad))
    top = torch.where(seen, s, torch.zeros_like(s)).abs().amax(-1, keepdim=True) if s.shape[1] else torch.zeros_like(m)
    spread = (q.abs() @ k.abs().mT * scale).amax(-1, keepdim=True) if s.shape[1] else torch.zeros_like(m)
    return out, size, top, spread


def tolerance(out, size, top, spread, d: int, n: int, dtype) -> torch.Tensor:
    """How far a correct kernel may be from ``out``, element by element.

    u = eps / 2 of the type.  The weights P are rounded to the type (u each)
    and divided by their own sum, so they are off by 2u in all: 2u * size.
    The output is rounded once: u |out|.  A score is a float32 sum of D exact
    products in some order (off by at most D 2^-24 of sum |q k| scale), scaled
    and shifted by the maximum (three roundings of numbers up to 2 top), and
    its exponential is off by 2^-22: the weights are off by e, numerator and
    denominator: 2 e size.  The float32 sums over n keys of one sign are off
    by at most n 2^-24 in the worst case and by sqrt(n) 2^-24 in practice;
    4 sqrt(n) 2^-24 is taken.  fp16 weights below 2^-33 of the largest are lost,
    n of them at most (n 2^-32 of the largest |v| in the row is above that).
    Numbers below the type's normal range are off by half its smallest step.
    """
    u = torch.finfo(dtype).eps / 2
    e = d * 2.0 ** -24 * spread + 6 * 2.0 ** -24 * top + 2.0 ** -22
    tol = (2 * u + 2 * e + 8 * math.sqrt(max(n, 1)) * 2.0 ** -24) * size + u * out.abs()
    if dtype == torch.float16:
        tol = tol + n * 2.0 ** -32 * size.amax(-1, keepdim=True) + 2.0 ** -25
    return torch.where(torch.isfinite(tol), tol * 1.01, torch.full_like(tol, math.inf))
