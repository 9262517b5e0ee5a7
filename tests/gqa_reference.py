"""Grouped-query attention written out in 64 bits, and how far 16-bit kernels may be off.

A rounding to 16 bits is off by at most u = eps / 2 relative to the value, and by u / sqrt(3) in the mean square. The kernels round,
beyond their result, the probabilities: the output's mean square error is u^2 / 3 sum_j p_j^2 v_j^2. Six times its root (the errors are
sums of many independent ones, or bounded by sqrt(3) of it where one term is all), the result's own rounding u |ref|, and
mla_reference.f32_part (f32 scores of n <= 576 terms, exponentials, sums over tokens) times sum_j p_j |v_j| bound the difference.
"""
import math

import torch

from mla_reference import f32_part, half_step, rotate, rotate_tol, softmax, tiny  # noqa: F401


def visible(pos, n, window=0, sinks=0):
    """[len(pos), n]: what queries at these positions see of n tokens."""
    j = torch.arange(n, device=pos.device)
    see = j <= pos[:, None]
    return see & ((j > pos[:, None] - window) | (j < sinks)) if window else see


def attend(q, k, v, pos, scale, u, window=0, sinks=0, hole=None):
    """q [nq, heads, dim] at positions pos over k, v [n, kv_heads, dim]: (out, tolerance), f64. hole [n]: tokens that are not seen.
    Values that are not finite count as 0 (they stand only where no query sees them)."""
    nq, heads, dim = q.shape
    kv_heads = k.shape[1]
    out = torch.zeros(nq, heads, dim, dtype=torch.float64, device=q.device)
    tol = torch.full_like(out, tiny(u))
    see = visible(pos, k.shape[0], window, sinks)
    if hole is not None:
        see = see & ~hole
    if not bool(see.any()):
        return out, tol
    for h in range(heads):
        x, y, w = q[:, h].double(), k[:, h * kv_heads // heads].double(), v[:, h * kv_heads // heads].double()
        w = torch.where(torch.isfinite(w), w, torch.zeros_like(w))
        p = softmax((scale * (x @ y.t())).masked_fill(~see, -math.inf))
        f32 = f32_part(torch.where(see, abs(scale) * (x.abs() @ y.abs().t()), torch.zeros_like(p)))
        o = p @ w
        out[:, h] = o
        tol[:, h] += u * o.abs() + 6 * u / math.sqrt(3) * (p.square() @ w.square()).sqrt() + f32 * (p @ w.abs())
    return out, tol
