"""Plain 64-bit forms of the quantised cache and of the two attentions, for their tests."""

from __future__ import annotations

import torch

F64 = torch.float64


def quantise(x: torch.Tensor, bits: int):
    """Rows ``x [..., 128]`` -> integer codes ``[..., 128]`` and scales bf16 ``[..., groups]``."""
    groups, most = (1, 127) if bits == 8 else (4, 7)
    g = x.float().reshape(*x.shape[:-1], groups, 128 // groups)
    top = g.abs().amax(-1)
    scale = (top / torch.full_like(top, most)).to(torch.bfloat16)
    scale = torch.where(scale.float() < torch.finfo(torch.float32).tiny, torch.zeros_like(scale), scale)
    scale = torch.where(torch.isfinite(top), scale, torch.full_like(scale, float("nan")))
    s = scale.float().unsqueeze(-1)
    code = torch.where(s > 0, torch.round(g / s).clamp(-most, most), torch.zeros_like(g))
    return code.flatten(-2).to(torch.int64), scale


def pack(code: torch.Tensor, bits: int) -> torch.Tensor:
    """Integer codes -> the stored bytes, one value at a time by the layout's definition."""
    if bits == 8:
        return (code + 128).to(torch.uint8)
    out = torch.zeros(*code.shape[:-1], 64, dtype=torch.int64)
    for d in range(128):
        run, place = d // 4, d % 4
        nibble = ((run % 8) * 4 + run // 8) * 4 + place
        out[..., nibble // 2] += (code[..., d] + 8) << (4 * (nibble % 2))
    return out.to(torch.uint8)


def restore(code: torch.Tensor, scale: torch.Tensor, bits: int) -> torch.Tensor:
    """Codes and scales -> float64 values."""
    size = 128 if bits == 8 else 32
    return code.to(F64) * scale.to(F64).repeat_interleave(size, -1)


def attention(q, k, v, scale):
    """Softmax attention ``q [G, 128]`` over ``k, v [n, 128]`` in float64; zeros without rows.  Also the weighted sums of
    the values' magnitudes, which the error bounds need."""
    q, k, v = q.to(F64), k.to(F64), v.to(F64)
    if k.shape[0] == 0:
        return torch.zeros_like(q), torch.zeros_like(q)
    w = torch.softmax(q @ k.T * scale, -1)
    return w @ v, w @ v.abs()


def output_bound(ref, weighted, dtype, score_error=0.0):
    """Largest error of an attention output.  A relative error ``e`` of every weight moves the quotient by at most
    ``2 e`` times the weighted sum of magnitudes; the output's own rounding is half a step of its type.
    bf16: the weights enter the products rounded to 16-bit floats, 2^-8 of them at most (half a step of bf16).
    float32: sums of up to a few thousand terms, each rounded to 2^-24, of which 2^-18 is a generous total."""
    if dtype == torch.bfloat16:
        return ref.abs() * 2.0 ** -8 + weighted * 2.0 * (2.0 ** -8 + score_error) + 1e-30
    return ref.abs() * 2.0 ** -24 + weighted * 2.0 * (2.0 ** -18 + score_error) + 1e-30
