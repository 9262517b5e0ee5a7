"""The latent-attention operators written out in 64 bits, and how far 16-bit kernels may be off.

A rounding to 16 bits is off by at most u = eps / 2 relative to the value, and by u / sqrt(3) in the mean
square. The kernels round, beyond their result, the probabilities; the latent query and the weighted latent (decode) are
held as two 16-bit numbers, off by at most u^2. With y_j the value that token j brings to an output (W_uv . c_j, or v_j) and Var_p the
variance over the probabilities, the output's mean square error is at most u^2 / 3 times

    sum_j p_j^2 y_j^2                                  the probabilities',
  + u^2 scale^2 Var_p(y) sum_i ql_i^2 Var_p(c_i)       the query's (|Cov_p(c_i, y)| <= sd_p(c_i) sd_p(y)),
  + u^2 sum_i o_i^2 W_uv[i]^2                          the weighted latent's.

Six times its root (the errors are sums of many independent ones, or bounded by sqrt(3) of it where one term is
all), the result's own rounding u |ref|, and (2^-16 + 96 2^-24 B) sum_j p_j |y_j| for the f32 work bound the difference: B is
the largest sum of the magnitudes of a score's terms, of which the f32 sum of n <= 576 terms is off by about sqrt(n) 2^-24 B
(four times that taken), and 2^-16 covers the exponentials and the sums over tokens (each good to a few 2^-22).
"""
import math

import torch


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rotate(x, pos, inv_freq, g, interleaved):
    """x [..., rope] f64 turned by pos (broadcast over the last dimension but one) * inv_freq."""
    a = pos.double()[..., None] * inv_freq.double()
    c, s = a.cos(), a.sin()
    if interleaved:
        x0, x1 = x[..., 0::2], x[..., 1::2]
    else:
        x0, x1 = x.chunk(2, -1)
    y0, y1 = g * (x0 * c - x1 * s), g * (x0 * s + x1 * c)
    return torch.stack([y0, y1], -1).flatten(-2) if interleaved else torch.cat([y0, y1], -1)


def rotate_tol(x, u, ref, interleaved):
    """The result's rounding, and 2^-20 (|x0| + |x1|): two f32 products and cosines good to 2^-22."""
    x = x.abs()
    if interleaved:
        n = (x[..., 0::2] + x[..., 1::2]).repeat_interleave(2, -1)
    else:
        n = (x.chunk(2, -1)[0] + x.chunk(2, -1)[1]).repeat(*[1] * (x.dim() - 1), 2)
    return u * ref.abs() * (1 + 2 ** -9) + 2.0 ** -20 * n + tiny(u)


def tiny(u):
    """Half a step of the smallest numbers: f16 values below 2^-14 have steps of 2^-24 (bf16's lie far below)."""
    return 2.0 ** -25 if u < 2 ** -9 else 0.0


def f32_part(magnitudes):
    return 2.0 ** -16 + 96 * 2.0 ** -24 * float(magnitudes.max())


def softmax(s):
    m = s.amax(-1, keepdim=True) if s.shape[-1] else s.new_zeros(s.shape[:-1] + (1,))
    p = torch.exp(s - torch.where(torch.isfinite(m), m, torch.zeros_like(m)))
    d = p.sum(-1, keepdim=True)
    return torch.where(d > 0, p / torch.where(d > 0, d, torch.ones_like(d)), torch.zeros_like(p))


def decode_row(q_nope, q_rope, kv_b, nope, c, kr, scale, u):
    """One query token [heads, ...] over its visible rows c [n, rank], kr [n, rope]; (out, tolerance), f64."""
    q_nope, q_rope, c, kr = (t.double() for t in (q_nope, q_rope, c, kr))
    if kv_b is not None:
        w_uk, w_uv = kv_b[:, :nope].double(), kv_b[:, nope:].double()
        ql = torch.bmm(q_nope[:, None].contiguous(), w_uk.contiguous())[:, 0]
    else:
        ql, w_uv = q_nope, None
    p = softmax(scale * (ql @ c.t() + q_rope @ kr.t()))
    f32 = f32_part(scale * (ql.abs() @ c.abs().t() + q_rope.abs() @ kr.abs().t()))
    o = p @ c
    var_c = (p @ c.square() - o.square()).clamp_min(0)
    from_q = (ql.square() * var_c).sum(-1) * scale ** 2 if kv_b is not None else 0 * ql[:, 0]
    if w_uv is None:
        out, var_y, size = o, var_c, p @ c.abs()
        from_p, from_o = p.square() @ c.square(), 0.0
    else:
        y = torch.matmul(w_uv.flatten(0, 1), c.t().contiguous()).view(w_uv.shape[0], w_uv.shape[1], -1)
        out = torch.bmm(w_uv.contiguous(), o[..., None].contiguous())[..., 0]
        var_y = ((y.square() * p[:, None]).sum(-1) - out.square()).clamp_min(0)
        from_p = (y.square() * p.square()[:, None]).sum(-1)
        from_o = torch.bmm(w_uv.square().contiguous(), o.square()[..., None].contiguous())[..., 0]
        size = (y.abs() * p[:, None]).sum(-1)
    rms = u / math.sqrt(3) * (from_p + u * u * (from_q[:, None] * var_y + from_o)).sqrt()
    return out, u * out.abs() + 6 * rms + f32 * size + tiny(u)


def prefill(q_nope, q_rope, kv, k_rope, nq, nk, nope, scale, u):
    """Ragged causal attention, f64: (out, tolerance)."""
    heads = q_nope.shape[1]
    out = torch.zeros(sum(nq), heads, kv.shape[2] - nope, dtype=torch.float64, device=kv.device)
    tol = torch.full_like(out, tiny(u))
    q0 = k0 = 0
    for a, b in zip(nq, nk):
        for h in range(heads if a and b else 0):
            k = torch.cat([kv[k0:k0 + b, h, :nope], k_rope[k0:k0 + b]], -1).double()
            q = torch.cat([q_nope[q0:q0 + a, h], q_rope[q0:q0 + a, h]], -1).double()
            seen = torch.arange(b, device=kv.device) <= torch.arange(a, device=kv.device)[:, None] + (b - a)
            s = (scale * (q @ k.t())).masked_fill(~seen, -math.inf)
            p = softmax(s)
            v = kv[k0:k0 + b, h, nope:].double()
            v = torch.where(torch.isfinite(v), v, torch.zeros_like(v))  # values that only masked places hold
            o = p @ v
            out[q0:q0 + a, h] = o
            f32 = f32_part(torch.where(seen, scale * (q.abs() @ k.abs().t()), torch.zeros_like(s)))
            tol[q0:q0 + a, h] += u * o.abs() + 6 * u / math.sqrt(3) * (p.square() @ v.square()).sqrt() + f32 * (p @ v.abs())
        q0, k0 = q0 + a, k0 + b
    return out, tol
