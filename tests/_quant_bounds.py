"""Error bounds of the attention over quantised rows, row by row and scale group by scale group, close enough that a lost tile
or a wrong scale falls outside."""

from __future__ import annotations

import torch

F64 = torch.float64


def attention_bound(q, k_code, k_scale, v_code, v_scale, bits, scale):
    """``q [G, 128]`` bf16 over ``n`` rows of integer codes ``[n, 128]`` and scales ``[n, groups]``, all on the CPU: the output
    in float64 and the largest error of the tensor-core path, both ``[G, 128]``.

    Score of a row.  The codes enter the products with an offset that the accumulators start without.  A partial sum of a scale
    group is at most ``M``: 1,152 (8 bits: 1,024 + 128) times the sum of the queries' magnitudes, in 4 bits 1,032 times that of
    the even components and 1,152 / 16 times that of the odd ones, whose queries are a sixteenth.  A product of 16 terms rounds
    (or cuts) it twice to 2^-22 of its size: 16 times in 8 bits, 4 times per group in 4 bits.  A query is a half float of
    at least 2^-25 (odd components of 4 bits: 2^-21) of the largest component, with 7 or 127 for the code; 2^9 times that where
    the largest is below 2^-20, since such queries are held nine places lower.  The key's scale and
    the softmax scale apply to all of it; scale, difference and exponential round the base-2 score to 2^-22 of its size.
    Weight times value scale is a half float: half a step is 2^-11 of it, or 2^-25 of the largest one of the component's group.
    Sums of n terms: 2^-24 of the sum of magnitudes each.  The output's own rounding: 2^-8 of it."""
    groups, size, most = (1, 128, 127) if bits == 8 else (4, 32, 7)
    n, qd = k_code.shape[0], q.to(F64)
    if n == 0:
        return torch.zeros_like(qd), torch.full_like(qd, 1e-30)
    ks, vs = k_scale.to(F64), v_scale.to(F64)
    k, v = k_code.to(F64) * ks.repeat_interleave(size, -1), v_code.to(F64) * vs.repeat_interleave(size, -1)
    z = qd @ k.T * scale
    w = torch.softmax(z, -1)
    out = w @ v
    a = qd.abs().view(-1, groups, size)
    if bits == 8:
        partial, times = 1152 * a.sum(-1), 16
    else:
        partial, times = 1032 * a[..., 0::2].sum(-1) + 72 * a[..., 1::2].sum(-1), 4
    top = a.amax((1, 2)).unsqueeze(-1)
    held = top * torch.where(top < 2.0 ** -20, 512.0, 1.0) * 2.0 ** (-25 if bits == 8 else -21)
    group = partial * times * 2.0 ** -22 + size * most * held                                         # [G, groups]
    e = group @ ks.T.abs() * abs(scale) + 2 * (z.abs() * 1.45 + 2) * 2.0 ** -22                       # [G, n]
    e = e + e * e                                          # exp(e) - 1, for e well below 1
    e = e + (w * e).sum(-1, keepdim=True)                  # the quotient's denominator moves too
    assert float(e.max()) < 0.5
    rounding = 2.0 ** -11 + (n + 64) * 2.0 ** -24
    small = (w.unsqueeze(-1) * vs.abs()).amax(1) * n * 2.0 ** -25 * most                              # [G, groups]
    bound = out.abs() * 2.0 ** -8 + (w * (e + rounding)) @ v.abs() + small.repeat_interleave(size, -1) + 1e-37
    return out, bound
