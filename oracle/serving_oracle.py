"""The serving operators restated on the CPU in 64 bits, from their definitions.

``rope``, ``quantize_rows`` / ``dequantize_rows`` and ``attention`` are what ``qk_norm_rope``, ``kv_cache_append`` /
``kv_cache_read`` and ``tree_attention`` compute before any rounding that is not part of the definition.
"""
from __future__ import annotations

import math

import torch

TOP = {torch.float8_e4m3fn: 448.0, torch.int8: 127.0}


def rope(x, positions, inv_freq, weight=None, eps=1e-6, interleaved=False):
    """(B, H, M, D) -> fp64; positions (M,) or (B, M)."""
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt(y.pow(2).mean(-1, keepdim=True) + eps) * weight.double()
    half = inv_freq.numel()
    t = positions.double().reshape(-1, 1, x.shape[2], 1) * inv_freq.double()
    c, s = torch.cos(t), torch.sin(t)
    out = y.clone()
    first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    a, b = y[..., first], y[..., second]
    out[..., first], out[..., second] = a * c - b * s, a * s + b * c
    return out


def _nearest_e4m3(u):
    """fp64 values of magnitude <= 448 rounded to the e4m3 grid, ties to even."""
    _, e = torch.frexp(u)  # |u| in [2^(e-1), 2^e): three fraction bits below the leading one, subnormals below 2^-6
    step = torch.ldexp(torch.ones_like(u), torch.clamp(e - 1, min=-6) - 3)
    return torch.round(u / step) * step


def quantize_rows(x, fmt):
    """Rows x (..., D) in fp16 or bf16 -> (fp64 codes, exponent bytes): the definition in ``kv_cache_append``."""
    y = x.double()
    fine = torch.isfinite(y).all(-1)
    y = torch.where(fine[..., None], y, 0.0)
    limit = torch.tensor(1.875 if fmt == torch.float8_e4m3fn else 1.96875).double() * (2.0 ** 15 if x.dtype == torch.float16 else 2.0 ** 127)
    top = y.abs().amax(-1) / TOP[fmt]
    mant, e = torch.frexp(top)  # top = mant * 2^e, mant in [0.5, 1)
    e = torch.where(mant == 0.5, e - 1, e)
    e = torch.where(top == 0, torch.full_like(e, -127), e.clamp(min=-127))
    u = torch.ldexp(torch.minimum(torch.maximum(y, -limit), limit), -e[..., None])
    codes = _nearest_e4m3(u) if fmt == torch.float8_e4m3fn else torch.round(u)
    return torch.where(fine[..., None], codes, 0.0), torch.where(fine, e + 127, 255).to(torch.uint8)


def dequantize_rows(codes, scale_bytes):
    """Codes (any type) and E8M0 bytes -> fp64 values."""
    f = torch.ldexp(torch.ones(scale_bytes.shape, dtype=torch.float64), scale_bytes.int() - 127)
    f = torch.where(scale_bytes == 255, math.nan, f)
    return codes.float().double() * f[..., None]


def attention(q, k, v, lengths, mask=None, scale=None):
    """fp64 (out, lse, weight): q (B,Hq,M,D), k and v (B,H,N,D) values; ``weight`` = sum_j p_ij |v_j| / sum_j p_ij, the scale of
    an error that is relative in p."""
    b, hq, m, d = q.shape
    h, n = k.shape[1], k.shape[2]
    scale = 1 / math.sqrt(d) if scale is None else scale
    out = torch.zeros(b, hq, m, d, dtype=torch.float64)
    wgt = torch.zeros_like(out)
    lse = torch.full((b, hq, m), -math.inf, dtype=torch.float64)
    for i in range(b):
        if int(lengths[i]) < 0:  # no positions, drafted ones neither
            continue
        have = min(int(lengths[i]), n)
        drafted = min(m, n - have)
        tree = torch.ones(m, m).tril().bool() if mask is None else (mask if mask.dim() == 2 else mask[i])
        for r in range(m):
            at = torch.cat([torch.arange(have), have + torch.nonzero(tree[r, :drafted]).flatten()])
            if at.numel() == 0:
                continue
            for g in range(hq):
                kk, vv = k[i, g // (hq // h), at].double(), v[i, g // (hq // h), at].double()
                s = kk @ q[i, g, r].double() * scale
                p = torch.softmax(s, 0)
                out[i, g, r], wgt[i, g, r], lse[i, g, r] = p @ vv, p @ vv.abs(), torch.logsumexp(s, 0)
    return out, lse, wgt
