"""Norm and rotation of queries and keys, stated in 64 bits (test infrastructure; see the package docstring).

Written from the definition: rows scaled to unit mean square, then turned in pairs.  Gradients come from autograd over this
statement; ``tests/test_oracle_cache.py`` holds them against differences.
"""
import torch


def turn(x, cos, sin, interleaved):
    """x (..., D), cos and sin (..., size / 2) that broadcast against x: the first ``size`` values turned in pairs."""
    half = cos.shape[-1]
    out = list(x.unbind(-1))
    for i in range(half):
        p, q = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        a, b = x[..., p], x[..., q]
        out[p] = a * cos[..., i] - b * sin[..., i]
        out[q] = b * cos[..., i] + a * sin[..., i]
    return torch.stack(out, -1)


def normalised(x, weight, eps):
    return x if weight is None else x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * weight


def norm_rotary(x, cos, sin, positions, weight, eps, interleaved):
    """x (B, H, T, D) float64 -> float64; positions (B, T); a position outside the tables turns by NaN."""
    rows = cos.shape[0]
    inside = ((positions >= 0) & (positions < rows))[..., None]
    at = positions.clamp(0, rows - 1).long()
    c, s = (torch.where(inside, t.double()[at], torch.nan)[:, None] for t in (cos, sin))
    return turn(normalised(x, weight, eps), c, s, interleaved)
