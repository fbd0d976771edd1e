"""The paged 8-bit cache in 64 bits, one sequence at a time: rotation, what an append leaves in a page, attention with a window and first tokens that stay visible."""
from __future__ import annotations

import math

import torch

Q_MAX = {"int8": 127.0, "fp8_e4m3": 448.0}
SCALE_MIN, MAGNITUDE = 2.0 ** -60, 2.0 ** 64


def rotated(x: torch.Tensor, first: int, rot_dims: int, base: float = 10000.0, pairing: str = "adjacent") -> torch.Tensor:
    """x f64 [rows, heads, dim] at positions first, first + 1, ..."""
    j = torch.arange(rot_dims // 2, dtype=torch.float64)
    angle = (first + torch.arange(x.shape[0], dtype=torch.float64))[:, None] * base ** (-2 * j / rot_dims)
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    out = x.clone()
    ia, ib = (slice(0, rot_dims, 2), slice(1, rot_dims, 2)) if pairing == "adjacent" else (slice(0, rot_dims // 2), slice(rot_dims // 2, rot_dims))
    a, b = x[..., ia], x[..., ib]
    out[..., ia], out[..., ib] = a * cos - b * sin, a * sin + b * cos
    return out


def nearest(y: torch.Tensor, dtype: str) -> torch.Tensor:
    """The code next to y (f64), as the number it is."""
    y = y.clamp(-Q_MAX[dtype], Q_MAX[dtype])
    return y.round() if dtype == "int8" else y.float().to(torch.float8_e4m3fn).double()


def append(codes: torch.Tensor, scale: float, older: int, x: torch.Tensor, dtype: str) -> tuple[torch.Tensor, float]:
    """One page and head: codes f64 [page_tokens, dim] of which the first `older` rows count, new rows x f64 [n, dim] behind them -> codes, scale."""
    codes = codes.clone()
    x = torch.where(x.abs() <= MAGNITUDE, x, torch.zeros_like(x))
    top = float(x.abs().max()) if x.numel() else 0.0
    need = max(top / Q_MAX[dtype], SCALE_MIN) if top > 0 else 0.0
    s = need
    if older and scale > 0:
        s, doublings = scale, 0
        while s < need:
            s, doublings = 2 * s, doublings + 1
        codes[:older] = nearest(codes[:older] * 2.0 ** -doublings, dtype)
    elif older:
        codes[:older] = 0
    codes[older:older + x.shape[0]] = nearest(x / s, dtype) if s > 0 else 0
    return codes, s


def visible(pos: torch.Tensor, keys: int, window: int, sinks: int) -> torch.Tensor:
    j = torch.arange(keys)
    seen = j <= pos[:, None]
    return seen & ((pos[:, None] - j < window) | (j < sinks)) if window else seen


def attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, top: torch.Tensor, first: int, scale: float, window: int = 0, sinks: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
    """q f64 [rows, q_heads, dim] at positions first ..; k, v f64 [tokens, kv_heads, dim]; top [tokens, kv_heads]: the largest value that a token's scale can stand for -> the
    result, and how far from it 32-bit scores and sums with weights in f16, rounded to bf16 at the end, may be:
    half a step of the result; on the weights' side half a step of f16 (2^-11) and twice the scores' error (a softmax weight moves by it, and so does their sum), with 2^-18 of
    the largest sum of |q k| and 2^-18 for the exponential, each many times what 32-bit sums of 128 terms are off by; and what f16 drops of small weights.  The weight of token j is held as
    p_j s_j / M, s_j its scale, M at most 2^-7 of the largest p_j s_j: off by 2^-25 at most where f16 has its least step of 2^-24.  It multiplies codes of up to top_j / s_j, so all of them
    together are off by 2^-25 * tokens * M * (largest code) <= 2^-32 * tokens * max(p_j top_j)."""
    rows, heads, _ = q.shape
    out, tol = torch.zeros_like(q), torch.zeros_like(q)
    seen = visible(torch.arange(first, first + rows), k.shape[0], window, sinks)
    for h in range(heads):
        kh, vh = k[:, h * k.shape[1] // heads], v[:, h * v.shape[1] // heads]
        s = (q[:, h] @ kh.T * scale).masked_fill(~seen, -math.inf)
        size = (q[:, h].abs() @ kh.abs().T * abs(scale)).masked_fill(~seen, 0).amax(1, keepdim=True)
        w = torch.nan_to_num((s - s.amax(1, keepdim=True)).exp())
        w = w / w.sum(1, keepdim=True).clamp_min(1e-300)
        out[:, h] = w @ vh
        dropped = 2.0 ** -32 * k.shape[0] * (w * top[:, h * v.shape[1] // heads]).amax(1, keepdim=True)
        tol[:, h] = 2.0 ** -8 * out[:, h].abs() + (2.0 ** -11 + 2.0 ** -17 * (1 + size)) * (w @ vh.abs()) + dropped
    return out, tol
