"""Rotary positions and the norm of query / key heads in 64 bits.

TEST INFRASTRUCTURE ONLY: the oracle of ``cast_rope`` and
``cast_qk_norm_rope``; nothing in the product imports it.  Written from the
formulas, with complex products for the turned pairs.
"""

from __future__ import annotations

import torch


def angles(positions: torch.Tensor, frequencies: torch.Tensor, axes=None) -> torch.Tensor:
    """positions ``[B,L]`` (``[B,L,3]`` with axes) -> float64 ``[B,L,pairs]``."""
    p = positions.to(torch.float64)
    f = frequencies.to(device=p.device, dtype=torch.float64)
    if axes is None:
        return p.unsqueeze(-1) * f
    out, at = [], 0
    for a, n in enumerate(axes):
        out.append(p[..., a:a + 1] * f[at:at + n])
        at += n
    return torch.cat(out, -1)


def turn(x: torch.Tensor, theta: torch.Tensor, interleaved: bool) -> torch.Tensor:
    """x float64 ``[B,L,H,D]``, theta ``[B,L,R/2]`` -> the first R values turned."""
    r = 2 * theta.shape[-1]
    first, second = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous())
    z = z * torch.polar(torch.ones_like(theta), theta).unsqueeze(2)
    y = x.clone()
    y[..., first], y[..., second] = z.real, z.imag
    return y


def pair_size(x: torch.Tensor, r: int, interleaved: bool) -> torch.Tensor:
    """``|a| + |b|`` of each value's pair (``|x|`` for those not turned), as x."""
    y = x.abs().clone()
    first, second = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    s = x[..., first].abs() + x[..., second].abs()
    y[..., first], y[..., second] = s, s
    return y


def norm(x: torch.Tensor, weight, eps: float) -> torch.Tensor:
    x = x.to(torch.float64)
    if weight is None:
        return x
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * weight.to(torch.float64)
