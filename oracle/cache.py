"""The cache operators in 64 bits, one sequence at a time: rows quantised to e4m3 with a power-of-two
scale, rows read back, and attention of a sequence's last tokens to its cache. No counterpart in the
reference, whose callers write their caches with torch."""

from __future__ import annotations

import math

import torch

from oracle.reference import gather_cache



def most(dtype: torch.dtype) -> float:
    """The largest magnitude of four significant bits that a type holds, which rows are held to."""
    return 1.875 * 2.0 ** (15 if dtype == torch.float16 else 127)


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Values (float64, after rounding) and scale exponents (int) of rows: the least e in [-126, 120] with
    m 2^-e <= 448 for the row's largest finite magnitude m (0 for m = 0), x 2^-e rounded to four
    significant bits, ties to even, on the grid of 2^-9 below 2^-6. Infinities become NaN.
    Magnitudes are held to most() first."""
    y = x.cpu().double()
    finite = torch.isfinite(y)
    y = y.clamp(-most(x.dtype), most(x.dtype))
    y = torch.where(finite, y, 0.0)
    top = y.abs().amax(dim=-1, keepdim=True)
    exponents = torch.zeros(top.shape, dtype=torch.float64)
    for index, m in enumerate(top.flatten().tolist()):
        if m > 0:
            fraction, power = math.frexp(m)  # m = fraction 2^power, fraction in [1/2, 1)
            e = power - 9 if fraction <= 0.875 else power - 8
            exponents.view(-1)[index] = min(max(e, -126), 120)
    scaled = y * torch.exp2(-exponents)
    step = torch.exp2(torch.frexp(scaled)[1].clamp(min=-5).double() - 4.0)
    values = torch.round(scaled / step) * step * torch.exp2(exponents)
    return torch.where(finite, values, math.nan), exponents.squeeze(-1).to(torch.int32)


def values(cache: torch.Tensor, scales: torch.Tensor | None) -> torch.Tensor:
    """What a cache's elements stand for, in float64 on the CPU."""
    cache = cache.cpu()
    if scales is None:
        return cache.double()
    exponents = scales.cpu().double() - 127.0
    return cache.float().double() * torch.exp2(exponents).unsqueeze(-1)


def rows_of(cache, scales, block_tables, b: int, length: int) -> torch.Tensor:
    """float64 values [length, H_kv, D] of a sequence's first rows."""
    cache = cache.cpu()
    tables = None if block_tables is None else block_tables.cpu()
    raw = cache.view(torch.uint8) if cache.dtype == torch.float8_e4m3fn else cache
    part = gather_cache(raw, tables, b, length).view(cache.dtype)
    if scales is None:
        return part.double()
    return values(part, gather_cache(scales.cpu(), tables, b, length))


def attention(q, k, v, positions, causal: bool, scale: float):
    """q [n, H, D], k and v [S, H_kv, D] in float64, positions [n] of the tokens. Returns o [n, H, D], lse
    [n, H], and what error bounds need: sum_j p_j |v_j| [n, H, D] and the largest scale sum_d |q_d k_jd|
    [n, H] over the visible keys."""
    n, heads, head_dim = q.shape
    keys, heads_kv = k.shape[:2]
    group = heads // heads_kv
    o, weight = torch.zeros(2, n, heads, head_dim, dtype=torch.float64)
    lse = torch.full((n, heads), -math.inf, dtype=torch.float64)
    size = torch.zeros((n, heads), dtype=torch.float64)
    hidden = torch.zeros((n, keys), dtype=torch.bool)
    if causal:
        hidden = torch.arange(keys)[None, :] > positions[:, None]
    seen = ~hidden.all(dim=-1)
    if keys == 0 or not seen.any():
        return o, lse, weight, size
    for h in range(heads):
        kh, vh = k[:, h // group], v[:, h // group]
        s = (q[:, h] @ kh.t() * scale).masked_fill(hidden, -math.inf)
        lse[:, h] = torch.logsumexp(s, dim=-1)
        p = torch.exp(s - lse[:, h, None].masked_fill(~seen[:, None], 0.0))
        o[:, h] = p @ vh
        weight[:, h] = p @ vh.abs()
        size[:, h] = (q[:, h].abs() @ kh.abs().t() * scale).masked_fill(hidden, 0.0).amax(dim=-1)
    return o, lse, weight, size
