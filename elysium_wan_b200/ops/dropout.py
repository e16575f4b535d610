"""Dropout on a residual branch, from a counter-based generator.

The mask is a function of (seed, stream, element) and is never stored: the
backward makes the same words again. ``word(e)`` of element e = row * d +
column is word e % 4 of the Philox4x32-10 block (Salmon et al., SC 2011) with
counter (e // 4, stream) under key seed, and an element is kept when its word
is at least round(p * 2**32). Every device type draws the same mask, and no
launch shape, stride or pipeline cut changes it; calls that must be
independent take different streams.
"""

from __future__ import annotations

import torch

from ._ext import ext

_LOW = 0xFFFFFFFF


def _check(p: float, seed: int, stream: int) -> None:
    if not 0.0 <= p < 1.0:
        raise ValueError(f"dropout probability {p} is not in [0, 1)")
    if not (0 <= seed < 1 << 64 and 0 <= stream < 1 << 64):
        raise ValueError("seed and stream are unsigned 64-bit numbers")


def dropout_words(n: int, seed: int, stream: int, device="cpu") -> torch.Tensor:
    """The first n words of a stream as int64 values in [0, 2**32)."""
    blk = torch.arange((n + 3) // 4, dtype=torch.int64, device=device)
    c0, c1 = blk & _LOW, blk >> 32
    c2, c3 = torch.full_like(blk, stream & _LOW), torch.full_like(blk, stream >> 32)
    k0, k1 = seed & _LOW, seed >> 32
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # 64-bit products modulo 2**64
        c0, c1, c2, c3 = (((b >> 32) & _LOW) ^ c1 ^ k0, b & _LOW,
                          ((a >> 32) & _LOW) ^ c3 ^ k1, a & _LOW)
        k0, k1 = (k0 + 0x9E3779B9) & _LOW, (k1 + 0xBB67AE85) & _LOW
    return torch.stack([c0, c1, c2, c3], 1).reshape(-1)[:n]


def dropout_add(x, resid, p: float, seed: int, stream: int, *, out_dtype=None):
    """resid + x * keep / (1 - p) over [rows, d]; resid None leaves the sum out.

    On the GPU x is bf16 or fp32 and resid any of bf16, fp16, fp32; rows may be
    strided. The sum is formed in fp32 and rounded once to out_dtype (x's
    unless given). A dropped element adds exactly 0, whatever x holds there.
    """
    _check(p, seed, stream)
    if x.is_cuda:
        return ext().dropout_add(x, resid, p, seed, stream, out_dtype)
    if x.dim() != 2 or (resid is not None and resid.shape != x.shape):
        raise ValueError("x must be [rows, d] and resid of the same shape")
    keep = dropout_words(x.numel(), seed, stream) >= min(round(p * 2**32), _LOW)
    y = torch.where(keep.view(x.shape), x.float() * (1.0 / (1.0 - p)), 0.0)
    if resid is not None:
        y = y + resid.float()
    return y.to(out_dtype or x.dtype)


def dropout_bwd(dy, p: float, seed: int, stream: int, *, out_dtype=None):
    """Gradient of x: dy * keep / (1 - p). The residual's gradient is dy itself."""
    return dropout_add(dy, None, p, seed, stream, out_dtype=out_dtype)
