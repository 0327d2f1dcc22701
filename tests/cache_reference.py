"""Plain 64-bit forms of the operators between the QKV and the O projection, on the CPU, and the error bounds that their tests use."""
from __future__ import annotations

import math

import torch

from breeze_tts_cpp_b200 import ops

RANGE = {ops.I8: 127.0, ops.FP8: 448.0}
F32_HALF = torch.finfo(torch.float32).eps / 2


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def least(dtype) -> float:
    """Half the spacing of the type's subnormal numbers."""
    info = torch.finfo(dtype)
    return info.tiny * info.eps / 2


def held(values: torch.Tensor, fmt: int) -> torch.Tensor:
    """One-byte storage as the numbers it stands for, in 64 bits."""
    return values.view(torch.int8 if fmt == ops.I8 else torch.float8_e4m3fn).to(torch.float64)


def turned(x: torch.Tensor, positions: torch.Tensor, turns: torch.Tensor, interleaved: bool, scale: float) -> torch.Tensor:
    """x [rows, heads, head_dim] in 64 bits."""
    half = turns.numel()
    angle = 2 * math.pi * torch.frac(positions.double()[:, None] * turns.double())
    c, n = scale * angle.cos()[:, None], scale * angle.sin()[:, None]
    y = x.clone()
    first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * c - b * n, b * c + a * n
    return y


def normed(x: torch.Tensor, weight: torch.Tensor | None, epsilon: float) -> torch.Tensor:
    if weight is None:
        return x
    return x / (x.square().mean(-1, keepdim=True) + epsilon).sqrt() * weight.double()


def attention(q, cache, pages, lengths, out, scale=None, offsets=None, prefix_pages=None, prefix_length=0):
    """What the operator's output buffer holds afterwards, in 64 bits, and a bound on its error for each element."""
    fmt, (_, kv_heads, page, head_dim) = cache.format, cache.keys.shape
    keys = held(cache.keys.cpu(), fmt) * cache.key_scales.cpu().double()[..., None]
    values = held(cache.values.cpu(), fmt) * cache.value_scales.cpu().double()[..., None]
    scale = head_dim**-0.5 if not scale else scale
    rows, width = q.shape
    group = width // head_dim // kv_heads
    want, bound = out.cpu().double().clone(), torch.zeros(rows, width, dtype=torch.float64)
    dtype = q.dtype
    offsets = list(range(rows + 1)) if offsets is None else offsets

    def rows_of(x, table, length):
        parts = [x[p] if 0 <= p < x.shape[0] else torch.full_like(x[0], math.nan) for p in table[: -(-length // page)]]
        return torch.cat(parts, 1)[:, :length] if parts else x.new_zeros(kv_heads, 0, head_dim)

    for b, length in enumerate(lengths):
        n = offsets[b + 1] - offsets[b]
        length = max(0, min(length, pages.shape[1] * page))
        k, v = (rows_of(x, pages[b].tolist(), length) for x in (keys, values))
        if prefix_pages is not None:
            k = torch.cat((rows_of(keys, prefix_pages.tolist(), prefix_length), k), 1)
            v = torch.cat((rows_of(values, prefix_pages.tolist(), prefix_length), v), 1)
        for i in range(n):
            row = offsets[b] + i
            seen = (prefix_length if prefix_pages is not None else 0) + max(0, length - n + i + 1)
            for h in range(kv_heads * group):
                x, at = q[row, h * head_dim: (h + 1) * head_dim].cpu().double(), slice(h * head_dim, (h + 1) * head_dim)
                if not seen:
                    want[row, at] = 0
                    continue
                score = k[h // group, :seen] @ x * scale
                weight = torch.softmax(score, 0)
                values_seen = v[h // group, :seen]
                want[row, at] = weight @ values_seen
                spread = weight @ values_seen.abs()
                # Weights are rounded to fp16 (half a step relative, and the subnormals' half spacing next to a largest weight of one).
                # Scores carry the rounding of their fp32 sums, products and exponents: a dozen half steps of the terms' magnitudes and
                # of the score itself in powers of two, which move a weight by that much relative to itself.
                magnitude = (k[h // group, :seen].abs() @ x.abs() * scale).max() * 1.4427 + 1
                moved = half_step(torch.float16) + 2 * 12 * F32_HALF * magnitude + 64 * F32_HALF
                most = values_seen.abs().max()
                bound[row, at] = (1 + half_step(dtype)) * (spread * moved + seen * least(torch.float16) * most) \
                    + want[row, at].abs() * half_step(dtype) + least(dtype)
    return want, bound


def check(got, want, bound, what=""):
    got = got.cpu().double()
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), f"{what}: NaN in other places"
    off = torch.where(nan, torch.zeros_like(got), (got - want).abs())
    limit = torch.where(nan, torch.ones_like(bound), bound)
    worst = (off / limit.clamp(min=1e-300)).max().item()
    assert (off <= limit).all(), f"{what}: error {worst:.3f} times its bound"
