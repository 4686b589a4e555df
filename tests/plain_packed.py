"""A paged cache of keys and values in 4 bits and attention over it, in plain float64: what the kernels are held against."""
from fractions import Fraction

import numpy as np
import torch

BLOCK = 64


def group_of(dim: int) -> int:
    return next(n for n in (64, 32, 16) if dim % n == 0)


def _nearest_even(x: Fraction) -> int:
    low = x.numerator // x.denominator
    rest = x - low
    return low + (1 if rest > Fraction(1, 2) or (rest == Fraction(1, 2) and low % 2) else 0)


def _bfloat16(x: Fraction) -> Fraction:
    """The nearest number of eight significant bits (of fewer below 2^-126), ties to even."""
    if x == 0:
        return x
    mag, e = abs(x), 0
    while mag >= Fraction(2) ** (e + 1):
        e += 1
    while mag < Fraction(2) ** e:
        e -= 1
    unit = Fraction(2) ** (max(e, -126) - 7)
    return (1 if x > 0 else -1) * _nearest_even(mag / unit) * unit


def quantise_group(numbers) -> tuple:
    """(step, zero, codes) of one group by exact rational arithmetic; NaN for a group that is not finite."""
    if not np.all(np.isfinite(numbers)):
        return float("nan"), float("nan"), [0] * len(numbers)
    x = [Fraction(float(v)) for v in numbers]
    zero = _bfloat16(min(x))
    step = max(_bfloat16((max(x) - zero) / 15), Fraction(0))
    if abs(zero) >= Fraction(2) ** 128 or max(x) - zero >= Fraction(2) ** 128 - Fraction(2) ** 103:
        return float("nan"), float("nan"), [0] * len(numbers)
    codes = [min(15, max(0, _nearest_even((v - zero) / step))) if step > 0 else 0 for v in x]
    return float(step), float(zero), codes


def quantise(rows: torch.Tensor, dim: int) -> tuple:
    """rows [T, heads·dim] → (codes [T, heads, dim] int64, pairs [T, heads, groups, 2] float64)."""
    T, G = rows.shape[0], group_of(dim)
    flat = rows.double().reshape(-1, G).numpy()
    codes, pairs = np.zeros(flat.shape, dtype=np.int64), np.zeros((flat.shape[0], 2))
    for i, numbers in enumerate(flat):
        step, zero, c = quantise_group(numbers)
        codes[i], pairs[i] = c, (step, zero)
    heads = rows.shape[1] // dim
    return torch.from_numpy(codes).view(T, heads, dim), torch.from_numpy(pairs).view(T, heads, dim // G, 2)


def values(codes: torch.Tensor, pairs: torch.Tensor) -> torch.Tensor:
    """float64 [..., dim] from codes [..., dim] and pairs [..., groups, 2]."""
    c = codes.double().view(*codes.shape[:-1], pairs.shape[-2], -1)
    return (pairs[..., 1:].double() + pairs[..., :1].double() * c).flatten(-2)


def unpacked(codes: torch.Tensor, pairs: torch.Tensor) -> torch.Tensor:
    """float64 values of a cache as it is stored: codes uint8 [..., dim/2], pairs bfloat16 [..., groups, 2]."""
    return values(torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2), pairs)


def attend(q, k, v, scale: float, window: int, pos: int) -> torch.Tensor:
    """One token: q [heads, dim], k and v [tokens, kv_heads, dim] of positions 0 …; float64 [heads, dim]."""
    first = max(0, pos - window + 1) if window > 0 else 0
    share = q.shape[0] // k.shape[1]
    out = []
    for h in range(q.shape[0]):
        s = (k[first:pos + 1, h // share] @ q[h]) * scale
        out.append(torch.softmax(s, dim=0) @ v[first:pos + 1, h // share])
    return torch.stack(out)
