"""Oracle of the paged cache (CPU, fp64): the 8-bit form of a block of tokens, the rotation, attention over a sequence.

Pinned by tests/test_oracle_paged.py.
"""

from __future__ import annotations

import math

import torch

E4M3_MAX = 448.0
BLOCK = 16
MIN_EXPONENT, MAX_EXPONENT = -118, 120
MIN_EXPONENT_FP16 = -15  # steps of codes below the normal ones are 2^-9 of the scale, of fp16 2^-24


def exponent_for(most: float, dtype: torch.dtype = torch.bfloat16) -> int:
    """The smallest e of those allowed with most <= 448 * 2^e."""
    e = MIN_EXPONENT
    if most > 0:
        m, x = math.frexp(most)  # most = m 2^x, 448 = 0.875 * 2^9
        e = x - 9 if m <= 0.875 else x - 8
    return max(MIN_EXPONENT_FP16 if dtype == torch.float16 else MIN_EXPONENT, min(MAX_EXPONENT, e))


def code_limit(e: int, dtype: torch.dtype) -> float:
    """The largest code of a block: 240 where 448 * 2^e passes the type (its largest number, rounded, would be infinite)."""
    return 240.0 if e >= (8 if dtype == torch.float16 else 120) else E4M3_MAX


def encode(x: torch.Tensor, e: int, dtype: torch.dtype) -> torch.Tensor:
    """The values that codes by the scale 2^e give for x (infinities and NaN: NaN)."""
    limit = code_limit(e, dtype)
    y = (x.double() * 2.0 ** -e).clamp(-limit, limit)
    y = torch.where(x.double().isfinite(), y, math.nan)
    return y.float().to(torch.float8_e4m3fn).double() * 2.0 ** e


def append_block(old: torch.Tensor, old_exponent: int, new: torch.Tensor, first: int, dtype: torch.dtype):
    """A block's values [16, D] and exponent after `new` [n, D] came to slots first .. first + n - 1."""
    finite = torch.where(new.double().isfinite(), new.double(), 0.0)
    e = exponent_for(float(finite.abs().max()) if finite.numel() else 0.0, dtype)
    if first > 0:
        e = max(e, old_exponent)
    values = old.clone()
    values[:first] = encode(old[:first], e, torch.bfloat16)
    values[first:first + len(new)] = encode(new, e, dtype)
    return values, e


def rotate(x: torch.Tensor, table: torch.Tensor, positions: torch.Tensor, interleaved: bool = False) -> torch.Tensor:
    """x [T, heads, D] with its first R elements rotated by rows of table [P, R] (cosines, sines)."""
    x, r = x.double().clone(), table.shape[1]
    cos, sin = (table.double()[positions][:, None, :].chunk(2, dim=-1))
    a, b = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    u, v = x[..., a].clone(), x[..., b].clone()
    x[..., a] = u * cos - v * sin
    x[..., b] = v * cos + u * sin
    return x


def attention(query: torch.Tensor, key: torch.Tensor, value: torch.Tensor, scale: float, dtype: torch.dtype):
    """(out, bound) of the last n = len(query) tokens of a sequence: query [n, H, D], key and value [L, Hkv, D].

    The bound counts: weights rounded to `dtype` and the result (half a step each), what fp32 loses of a score (D products
    summed, the scale, the exponential) and of sums over L keys, and fp16 weights below its normal numbers: these are rounded
    with the largest at 2^7, by half of 2^-24.
    """
    n, heads, d = query.shape
    length, hkv, _ = key.shape
    half = torch.finfo(dtype).eps / 2
    q, k, v = query.double(), key.double(), value.double()
    out = torch.zeros(n, heads, d, dtype=torch.float64)
    bound = torch.zeros_like(out)
    if length == 0:
        return out, bound
    hidden = torch.arange(length) > (length - n + torch.arange(n))[:, None]
    for h in range(heads):
        kh, vh = k[:, h // (heads // hkv)], v[:, h // (heads // hkv)]
        z = (q[:, h] @ kh.T * scale).masked_fill(hidden, -math.inf)
        p = torch.nan_to_num(torch.softmax(z, dim=-1))
        seen = torch.where(hidden[..., None], 0.0, vh)  # what a row does not see takes no part, NaN neither
        out[:, h] = (p[..., None] * seen).sum(dim=1)
        size = (p[..., None] * seen.abs()).sum(dim=1)
        score = ((q[:, h].abs() @ kh.abs().T) * abs(scale)).masked_fill(hidden, 0.0).amax(dim=-1, keepdim=True)
        loss = (d + 8) * 2.0 ** -24 * score + (length + 16) * 2.0 ** -24 + 2.0 ** -21
        bound[:, h] = size * (half + 2 * loss) + out[:, h].abs() * half
        if dtype == torch.float16:
            bound[:, h] += length * 2.0 ** -32 * seen.abs().amax(dim=1) + 2.0 ** -25
    return out, bound
