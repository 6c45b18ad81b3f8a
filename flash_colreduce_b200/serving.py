"""What a serving program runs around the column reduction.

``qk_norm_rope`` makes the queries and keys that :func:`flash_colreduce` takes, ``kv_cache_append`` and
``kv_cache_read`` keep keys and values in a cache of 16 or 8 bits and read them back (whole, or at the positions that
:func:`topk_columns` selected), and ``tree_attention`` lets drafted tokens -- or the one token of plain decoding --
attend that cache.  The reference has no counterpart; its README.md:9 names the token pruning these belong to.

All of it is forward only: inputs that require a gradient are refused while gradients are recorded, and inputs that carry a
tangent of forward-mode differentiation always.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional, Tuple

import torch
from torch.autograd import forward_ad

from . import _native as nat
from .op import _DTYPE_CODES, _debug_sync, _on_device

__all__ = ["qk_norm_rope", "kv_cache_append", "kv_cache_read", "tree_attention"]

_increment_version = torch.autograd.graph.increment_version
_INDEX_BITS = {torch.int32: 32, torch.int64: 64}
_FORMATS = {torch.float16: nat.FCR_KV_16BIT, torch.bfloat16: nat.FCR_KV_16BIT, torch.float8_e4m3fn: nat.FCR_KV_FP8,
            torch.int8: nat.FCR_KV_INT8}
_SCALE_DTYPES = (torch.float8_e8m0fnu, torch.uint8)


def _check_devices(device: torch.device, **tensors) -> None:
    for name, x in tensors.items():
        if x is None:
            continue
        if not x.is_cuda:
            raise ValueError(f"{name} must be on a CUDA device.")
        if x.device != device:
            raise ValueError(f"All tensors must be on one device; got {name} on {x.device}, not {device}.")


def _derivatives() -> bool:
    """Whether gradients are recorded or tangents may be carried (no_grad does not end those)."""
    return torch.is_grad_enabled() or forward_ad._current_level >= 0


def _check_no_grad(what: str, *tensors) -> None:
    given = [x for x in tensors if x is not None]
    if torch.is_grad_enabled() and any(x.requires_grad for x in given):
        raise RuntimeError(f"{what} has no backward pass: call it under torch.no_grad().")
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(x).tangent is not None for x in given):
        raise RuntimeError(f"{what} has no forward-mode derivative: pass the primal (torch.autograd.forward_ad.unpack_dual).")


_MAX_ROWS = 2 ** 30  # rows, positions and heads are counted in 32 bits


def _check_sizes(**counts) -> None:
    for name, count in counts.items():
        if count > _MAX_ROWS:
            raise ValueError(f"{count} {name.replace('_', ' ')} exceed {_MAX_ROWS}.")


def _rows(x: torch.Tensor) -> torch.Tensor:
    """``x`` with an innermost stride of 1 (a copy when it has another)."""
    return x if x.stride(-1) == 1 or x.shape[-1] == 1 and x.is_contiguous() else x.contiguous()


# What a call's signature (shapes, strides, types, devices, options; no data, no addresses) comes to.  Small calls are bound
# by the host, so that a signature is checked once.
_ROPE_CACHE: dict = {}
_APPEND_CACHE: dict = {}
_READ_CACHE: dict = {}
_TREE_CACHE: dict = {}


def _keep(cache: dict, signature, value) -> None:
    if len(cache) > 4096:
        cache.clear()
    cache[signature] = value


def _vector_signature(x: Optional[torch.Tensor]):
    return None if x is None else (x.shape, x.stride(), x.dtype, x.get_device())


def qk_norm_rope(
    query: torch.Tensor,
    key: torch.Tensor,
    positions: torch.Tensor,
    inv_freq: torch.Tensor,
    q_weight: Optional[torch.Tensor] = None,
    k_weight: Optional[torch.Tensor] = None,
    eps: float = 1e-6,
    interleaved: bool = False,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """RMS norm of every head's queries and keys and rotation by position, in one kernel.

    ``y = x * rsqrt(mean(x^2) + eps) * weight`` over the head dimension (without a weight ``y = x``), then the pairs
    ``(i, i + R/2)`` -- or ``(2 i, 2 i + 1)`` with ``interleaved`` -- of the first ``R = 2 * len(inv_freq)`` dimensions are
    rotated by ``position * inv_freq[i]``.  Computed in fp32, the angle in fp64, and rounded once; a row whose sum of squares
    passes fp32's range is normed to zeros.  No more than 2^30 tokens, heads or sequences.

    Args:
        query: (B, Hq, M, D) fp16, bf16 or fp32 CUDA tensor with D <= 256; any strides with innermost 1, e.g. a view of
            a fused projection's (B, M, heads, D) output (other innermost strides are copied).
        key: (B, Hk, M, D), same type and device.
        positions: (M,) or (B, M) int32 or int64.
        inv_freq: (R / 2,) fp32, R <= D.
        q_weight, k_weight: (D,) of the inputs' type or fp32 (both of one type), or None for no norm.

    Returns:
        ``(query, key)``, new contiguous tensors of the inputs' type.
    """
    if _derivatives():
        _check_no_grad("qk_norm_rope", query, key, q_weight, k_weight, inv_freq)
    eps, interleaved = float(eps), bool(interleaved)  # (plain values: a signature must not hold a tensor)
    signature = (query.shape, query.stride(), query.dtype, query.get_device(), key.shape, key.stride(), key.dtype, key.get_device(), positions.shape,
                 positions.stride(), positions.dtype, positions.get_device(), inv_freq.shape, inv_freq.is_contiguous(), inv_freq.dtype, inv_freq.get_device(),
                 _vector_signature(q_weight), _vector_signature(k_weight), eps, interleaved)
    problem = _ROPE_CACHE.get(signature)
    if problem is None:
        problem, query, key, inv_freq, q_weight, k_weight = _plan_rope(signature, query, key, positions, inv_freq, q_weight, k_weight, eps,
                                                                       interleaved)
    b, hq, m, d = query.shape
    dtype, device = query.dtype, query.device
    q_out = torch.empty((b, hq, m, d), dtype=dtype, device=device)
    k_out = torch.empty((b, problem.Hk, m, d), dtype=dtype, device=device)
    if problem.B * problem.M * problem.D * (problem.Hq + problem.Hk) == 0:
        return q_out, k_out
    index = device.index
    with _on_device(index):
        rc = nat.lib.fcr_qk_norm_rope(C.byref(problem), query.data_ptr(), key.data_ptr(), positions.data_ptr(), inv_freq.data_ptr(),
                                      None if q_weight is None else q_weight.data_ptr(),
                                      None if k_weight is None else k_weight.data_ptr(), q_out.data_ptr(), k_out.data_ptr(),
                                      torch._C._cuda_getCurrentRawStream(index))
        if rc:
            nat.check(rc, "fcr_qk_norm_rope")
    return q_out, k_out


def _plan_rope(signature, query, key, positions, inv_freq, q_weight, k_weight, eps, interleaved):
    """Checks a call of ``qk_norm_rope`` and describes it; the description is kept when the tensors go in as they lie."""
    if query.dim() != 4 or key.dim() != 4 or any(query.shape[i] != key.shape[i] for i in (0, 2, 3)):
        raise ValueError(f"query and key must be (B, H, M, D) with the same B, M and D; got {tuple(query.shape)} and {tuple(key.shape)}.")
    if query.dtype != key.dtype or query.dtype not in _DTYPE_CODES:
        raise TypeError(f"qk_norm_rope takes fp16, bf16 or fp32 tensors of one dtype; got query {query.dtype}, key {key.dtype}.")
    b, hq, m, d = query.shape
    hk = key.shape[1]
    _check_sizes(sequences=b, tokens=m, heads=hq + hk)
    if d > 256:
        raise ValueError(f"Head dimension {d} exceeds 256.")
    if inv_freq.dtype != torch.float32 or inv_freq.dim() != 1 or 2 * inv_freq.shape[0] > d:
        raise ValueError(f"inv_freq must be fp32 of shape (R / 2,) with R <= {d}; got {inv_freq.dtype} {tuple(inv_freq.shape)}.")
    if positions.dtype not in _INDEX_BITS or tuple(positions.shape) not in ((m,), (b, m)):
        raise ValueError(f"positions must be int32 or int64 of shape ({m},) or ({b}, {m}); got {positions.dtype} {tuple(positions.shape)}.")
    weights = [w for w in (q_weight, k_weight) if w is not None]
    for w in weights:
        if w.dim() != 1 or w.shape[0] != d or w.dtype not in (query.dtype, torch.float32) or w.dtype != weights[0].dtype:
            raise ValueError(f"weights must be ({d},) of {query.dtype} or fp32, both of one type; got {w.dtype} {tuple(w.shape)}.")
    _check_devices(query.device, query=query, key=key, positions=positions, inv_freq=inv_freq, q_weight=q_weight,
                   k_weight=k_weight)
    given = (query, key, inv_freq, q_weight, k_weight)
    used = (_rows(query), _rows(key), inv_freq.contiguous(), *(None if w is None else w.contiguous() for w in (q_weight, k_weight)))
    query, key, inv_freq = used[:3]
    p = nat.Rope(b, hq, hk, m, d, 2 * inv_freq.shape[0], (*query.stride()[:3], 1), (*key.stride()[:3], 1),
                 _DTYPE_CODES[query.dtype], _DTYPE_CODES[weights[0].dtype] if weights else 0, int(interleaved),
                 _INDEX_BITS[positions.dtype], (positions.stride(0) if positions.dim() == 2 else 0, positions.stride(-1)),
                 eps)
    if all(x is y for x, y in zip(given, used)):
        _keep(_ROPE_CACHE, signature, p)
    return (p, *used)


def _cache_problem(key_cache, value_cache, key_scales, value_scales, dtype) -> nat.KvCache:
    """Checks a cache's tensors against one another and describes them; ``dtype``: the type of the values it holds."""
    if key_cache.dim() != 4 or key_cache.shape != value_cache.shape:
        raise ValueError(f"key_cache and value_cache must be (B, H, N, D) of one shape; got {tuple(key_cache.shape)} and {tuple(value_cache.shape)}.")
    if key_cache.dtype != value_cache.dtype or key_cache.dtype not in _FORMATS:
        raise TypeError(f"a cache is fp16, bf16, float8_e4m3fn or int8; got key_cache {key_cache.dtype}, value_cache {value_cache.dtype}.")
    if dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"a cache holds fp16 or bf16 values; got {dtype}.")
    fmt = _FORMATS[key_cache.dtype]
    b, h, n, d = key_cache.shape
    _check_sizes(positions=n, heads_of_sequences=b * h)
    if d > 256:
        raise ValueError(f"Head dimension {d} exceeds 256.")
    if fmt == nat.FCR_KV_16BIT:
        if key_cache.dtype != dtype:
            raise TypeError(f"a 16-bit cache holds values of its own type {key_cache.dtype}, not {dtype}.")
        if key_scales is not None or value_scales is not None:
            raise ValueError("a 16-bit cache has no scales.")
        ss = ((0, 0, 0), (0, 0, 0))
    else:
        for name, s in (("key_scales", key_scales), ("value_scales", value_scales)):
            if s is None or s.dtype not in _SCALE_DTYPES or s.shape != (b, h, n):
                raise ValueError(f"an 8-bit cache needs {name} of float8_e8m0fnu (or their bytes as uint8) and shape ({b}, {h}, {n})"
                                 + ("." if s is None else f"; got {s.dtype} {tuple(s.shape)}."))
        ss = (key_scales.stride(), value_scales.stride())
    if d > 1 and (key_cache.stride(3) != 1 or value_cache.stride(3) != 1):
        raise ValueError("the innermost stride of a cache must be 1.")
    return nat.KvCache(b, h, n, d, fmt, _DTYPE_CODES[dtype], (*key_cache.stride()[:3], 1), (*value_cache.stride()[:3], 1), *ss)


def _lengths(name, x, b):
    if x.dtype not in _INDEX_BITS or tuple(x.shape) != (b,):
        raise ValueError(f"{name} must be int32 or int64 of shape ({b},); got {x.dtype} {tuple(x.shape)}.")
    return x.contiguous()


def _address(x: Optional[torch.Tensor]):
    return None if x is None else x.data_ptr()


def kv_cache_append(
    key: torch.Tensor,
    value: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    lengths: torch.Tensor,
    key_scales: Optional[torch.Tensor] = None,
    value_scales: Optional[torch.Tensor] = None,
    counts: Optional[torch.Tensor] = None,
) -> None:
    """Writes M new tokens of every sequence into a cache, in place, quantising them when it holds 8 bits.

    Token ``m`` of sequence ``b`` goes to position ``lengths[b] + m``; with ``counts`` only the first ``counts[b]`` tokens
    are written.  Tokens of a negative length or beyond the capacity are left out, and positions that are not written
    keep what they held.  ``lengths`` stays as it is: a program adds what it appended (or what was accepted of it).

    An 8-bit cache holds, per row (a token's head of K or V), codes and one power-of-two scale ``2^e``: ``e`` is the
    least exponent (at least -127) for which the row's largest magnitude is at most ``448 * 2^e`` (float8_e4m3fn) or
    ``127 * 2^e`` (int8), a code is ``x / 2^e`` rounded to nearest even.  Values that would read back as an infinity are
    clamped to the largest that does not.  A row with a NaN or an infinity reads back as NaN.  A cache has at most 2^30
    positions, and as many heads of all sequences together.

    Args:
        key, value: (B, H, M, D) fp16 or bf16, D <= 256; any strides with innermost 1 (others are copied).
        key_cache, value_cache: (B, H, N, D) of the same type (plain copies), float8_e4m3fn or int8; they overlap neither
            each other nor the inputs.
        lengths: (B,) int32 or int64.
        key_scales, value_scales: (B, H, N) float8_e8m0fnu or uint8, for 8-bit caches.
        counts: (B,) of the type of ``lengths``, or None.
    """
    if _derivatives():
        _check_no_grad("kv_cache_append", key, value, key_cache, value_cache)
    signature = (key.shape, key.stride(), key.dtype, key.get_device(), value.shape, value.stride(), value.dtype, value.get_device(), key_cache.shape,
                 key_cache.stride(), key_cache.dtype, key_cache.get_device(), value_cache.shape, value_cache.stride(), value_cache.dtype,
                 value_cache.get_device(), lengths.shape, lengths.is_contiguous(), lengths.dtype, lengths.get_device(), _vector_signature(key_scales),
                 _vector_signature(value_scales), _vector_signature(counts))
    hit = _APPEND_CACHE.get(signature)
    if hit is None:
        hit, key, value, lengths, counts = _plan_append(signature, key, value, key_cache, value_cache, lengths, key_scales, value_scales,
                                                        counts)
    if hit == 0:  # nothing to write
        return
    problem, key_strides, value_strides, m, index_bits, index = hit
    with _on_device(index):
        rc = nat.lib.fcr_kv_append(C.byref(problem), key_cache.data_ptr(), value_cache.data_ptr(), _address(key_scales),
                                   _address(value_scales), key.data_ptr(), key_strides, value.data_ptr(), value_strides, m,
                                   lengths.data_ptr(), _address(counts), index_bits, torch._C._cuda_getCurrentRawStream(index))
        if rc:
            nat.check(rc, "fcr_kv_append")
    # autograd cannot see a write through a pointer: a cache that an operation saved for its backward pass must not change unnoticed
    _increment_version([x for x in (key_cache, value_cache, key_scales, value_scales) if x is not None])


def _plan_append(signature, key, value, key_cache, value_cache, lengths, key_scales, value_scales, counts):
    """Checks a call of ``kv_cache_append`` and describes it (0: nothing to write), as ``_plan_rope`` does."""
    if key.dtype != value.dtype:
        raise TypeError(f"key and value must be of one dtype; got {key.dtype} and {value.dtype}.")
    problem = _cache_problem(key_cache, value_cache, key_scales, value_scales, key.dtype)
    b, h, n, d = key_cache.shape
    if key.dim() != 4 or key.shape != value.shape or key.shape[:2] != (b, h) or key.shape[3] != d:
        raise ValueError(f"key and value must be ({b}, {h}, M, {d}); got {tuple(key.shape)} and {tuple(value.shape)}.")
    _check_sizes(tokens=key.shape[2])
    for name, x in (("key_cache", key_cache), ("value_cache", value_cache), ("key_scales", key_scales), ("value_scales", value_scales)):
        if x is not None and any(x.shape[i] > 1 and x.stride(i) == 0 for i in range(3)):
            raise ValueError(f"{name} is written: it cannot be an expanded tensor.")
    given = (key, value, lengths, counts)
    lengths = _lengths("lengths", lengths, b)
    if counts is not None:
        if counts.dtype != lengths.dtype:
            raise ValueError(f"counts must be of the type of lengths ({lengths.dtype}); got {counts.dtype}.")
        counts = _lengths("counts", counts, b)
    _check_devices(key.device, key=key, value=value, key_cache=key_cache, value_cache=value_cache, lengths=lengths,
                   key_scales=key_scales, value_scales=value_scales, counts=counts)
    if key.numel() == 0 or n == 0:
        return 0, key, value, lengths, counts
    key, value = _rows(key), _rows(value)
    hit = (problem, nat.strides4(key.stride()), nat.strides4(value.stride()), key.shape[2], _INDEX_BITS[lengths.dtype], key.device.index)
    if all(x is y for x, y in zip(given, (key, value, lengths, counts))):
        _keep(_APPEND_CACHE, signature, hit)
    return hit, key, value, lengths, counts


def kv_cache_read(
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    key_scales: Optional[torch.Tensor] = None,
    value_scales: Optional[torch.Tensor] = None,
    positions: Optional[torch.Tensor] = None,
    n: Optional[int] = None,
    dtype: Optional[torch.dtype] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Keys and values of a cache in 16 bits: the first ``n`` positions, or the ones that ``positions`` names.

    ``positions`` (B, H, n) int32 or int64 selects per head -- the indices :func:`topk_columns` returns, say; a
    position outside the cache reads as zeros.  Without it the first ``n`` positions (all of them by default) are read.
    Reading in the type that the rows were written from is exact; another ``dtype`` rounds.

    Args:
        key_cache, value_cache, key_scales, value_scales: as for :func:`kv_cache_append`.
        dtype: torch.float16 or torch.bfloat16; a 16-bit cache is read in its own type, an 8-bit one as bf16 by default.

    Returns:
        ``(key, value)``, contiguous (B, H, n, D): what :func:`flash_colreduce` takes as keys.
    """
    if _derivatives():
        _check_no_grad("kv_cache_read", key_cache, value_cache)
    if n is not None:
        n = int(n)
    signature = (key_cache.shape, key_cache.stride(), key_cache.dtype, key_cache.get_device(), value_cache.shape, value_cache.stride(),
                 value_cache.dtype, value_cache.get_device(), _vector_signature(key_scales), _vector_signature(value_scales),
                 _vector_signature(positions), n, dtype)
    hit = _READ_CACHE.get(signature)
    if hit is None:
        hit, positions = _plan_read(signature, key_cache, value_cache, key_scales, value_scales, positions, n, dtype)
    problem, shape, dtype, index_bits, device = hit
    k_out = torch.empty(shape, dtype=dtype, device=device)
    v_out = torch.empty(shape, dtype=dtype, device=device)
    if k_out.numel() == 0:
        return k_out, v_out
    if problem.N == 0:
        return k_out.zero_(), v_out.zero_()
    index = device.index
    with _on_device(index):
        rc = nat.lib.fcr_kv_read(C.byref(problem), key_cache.data_ptr(), value_cache.data_ptr(), _address(key_scales),
                                 _address(value_scales), _address(positions), index_bits, shape[2], k_out.data_ptr(), v_out.data_ptr(),
                                 torch._C._cuda_getCurrentRawStream(index))
        if rc:
            nat.check(rc, "fcr_kv_read")
    return k_out, v_out


def _plan_read(signature, key_cache, value_cache, key_scales, value_scales, positions, n, dtype):
    """Checks a call of ``kv_cache_read`` and describes it, as ``_plan_rope`` does."""
    if dtype is None:
        dtype = key_cache.dtype if key_cache.dtype in (torch.float16, torch.bfloat16) else torch.bfloat16
    problem = _cache_problem(key_cache, value_cache, key_scales, value_scales, dtype)
    b, h, cap, d = key_cache.shape
    given = positions
    if positions is not None:
        if positions.dtype not in _INDEX_BITS or positions.dim() != 3 or positions.shape[:2] != (b, h):
            raise ValueError(f"positions must be int32 or int64 of shape ({b}, {h}, n); got {positions.dtype} {tuple(positions.shape)}.")
        if n is not None and n != positions.shape[2]:
            raise ValueError(f"n = {n} and positions of shape {tuple(positions.shape)} disagree.")
        n = positions.shape[2]
        _check_sizes(positions=n)
        positions = positions.contiguous()
    else:
        n = cap if n is None else n
        if not 0 <= n <= cap:
            raise ValueError(f"n = {n} must lie in [0, {cap}].")
    _check_devices(key_cache.device, key_cache=key_cache, value_cache=value_cache, key_scales=key_scales,
                   value_scales=value_scales, positions=positions)
    hit = (problem, (b, h, n, d), dtype, 64 if positions is None else _INDEX_BITS[positions.dtype], key_cache.device)
    if positions is given:
        _keep(_READ_CACHE, signature, hit)
    return hit, positions


def tree_attention(
    query: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    lengths: torch.Tensor,
    tree_mask: Optional[torch.Tensor] = None,
    scale: Optional[float] = None,
    key_scales: Optional[torch.Tensor] = None,
    value_scales: Optional[torch.Tensor] = None,
    return_lse: bool = False,
):
    """Attention of M drafted tokens of every sequence over a KV cache; M = 1 is plain decoding.

    The drafted tokens' own keys and values lie in the cache at positions ``lengths[b] .. lengths[b] + M - 1``
    (:func:`kv_cache_append` with the same ``lengths`` puts them there).  Every token attends the ``lengths[b]``
    positions before them and, among the drafted tokens, those its row of ``tree_mask`` names; without a mask they
    are a chain (token ``m`` attends drafted tokens ``j <= m``).  Positions beyond the capacity do not exist, and a sequence
    of negative length has none, drafted ones neither.  A row that attends nothing returns 0 (and a log-sum-exp of -inf).  What masked and unwritten positions hold does not
    matter, NaN and infinities included.

    Args:
        query: (B, Hq, M, D) fp16 or bf16, M <= 256, D <= 128; strides that are not multiples of 16 bytes are copied.
        key_cache, value_cache: (B, H, N, D), Hq a multiple of H (query head ``h`` reads cache head ``h // (Hq // H)``);
            of ``query``'s type with D a multiple of 8, or float8_e4m3fn / int8 with D a multiple of 16.  Base addresses
            and strides are multiples of 16 bytes.
        lengths: (B,) int32 or int64, on the GPU: a captured graph may be replayed with other values.
        tree_mask: (M, M), (1, M, M) or (B, M, M) bool, or None.
        scale: softmax scale, finite (up to 2.3e38), default ``1 / sqrt(D)``.
        key_scales, value_scales: (B, H, N) float8_e8m0fnu or uint8, for 8-bit caches.

    Returns:
        (B, Hq, M, D) of ``query``'s type, and with ``return_lse`` also the fp32 (B, Hq, M) natural log-sum-exp of
        every row's scaled scores.  Run-to-run results are bitwise identical.

    Scores, sums and accumulators are fp32.  Cached values are taken in ``query``'s type, and the softmax weights are rounded
    to that type once before they multiply them: by half a step, 2^-8 of a weight in bf16, 2^-11 in fp16 (there at least 2^-32
    of the row's sum per key).  An 8-bit cache takes about half the memory of a 16-bit one; for single tokens the attention is up to 7 %
    faster over it, for drafted ones slower (by 8 % with 16 rows per cache head, up to 36 % with 128).
    """
    if _derivatives():
        _check_no_grad("tree_attention", query, key_cache, value_cache)
    if scale is not None:
        scale = float(scale)
    signature = (query.shape, query.stride(), query.dtype, query.get_device(), key_cache.shape, key_cache.stride(), key_cache.dtype,
                 key_cache.get_device(), value_cache.shape, value_cache.stride(), value_cache.dtype, value_cache.get_device(), lengths.shape,
                 lengths.is_contiguous(), lengths.dtype, lengths.get_device(), _vector_signature(tree_mask), scale, _vector_signature(key_scales),
                 _vector_signature(value_scales))
    hit = _TREE_CACHE.get(signature)
    if hit is None or query.data_ptr() % 16:
        hit, query, lengths, tree_mask = _plan_tree(signature, query, key_cache, value_cache, lengths, tree_mask, scale, key_scales,
                                                    value_scales)
    problem, tree, shape, dtype, device, ws_bytes = hit
    out = torch.empty(shape, dtype=dtype, device=device)
    lse = torch.empty(shape[:3], dtype=torch.float32, device=device) if return_lse else None
    if ws_bytes == 0:  # no rows, or no positions that they could attend
        out.zero_()
        return (out, lse.fill_(-math.inf)) if return_lse else out
    index = device.index
    with _on_device(index):
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=device)
        stream = torch._C._cuda_getCurrentRawStream(index)
        rc = nat.lib.fcr_tree_attention(C.byref(problem), C.byref(tree), query.data_ptr(), key_cache.data_ptr(),
                                        value_cache.data_ptr(), _address(key_scales), _address(value_scales),
                                        lengths.data_ptr(), _address(tree_mask), out.data_ptr(), _address(lse), ws.data_ptr(),
                                        ws_bytes, stream)
        if rc == nat.FCR_ERR_UNSUPPORTED:
            raise ValueError(nat.last_error())
        if rc:
            nat.check(rc, "fcr_tree_attention")
        if _debug_sync() and not torch.cuda.is_current_stream_capturing():
            nat.check(nat.lib.fcr_read_device_status(ws.data_ptr(), stream, None), "fcr_tree_attention (device)")
    return (out, lse) if return_lse else out


def _plan_tree(signature, query, key_cache, value_cache, lengths, tree_mask, scale, key_scales, value_scales):
    """Checks a call of ``tree_attention`` and describes it (no workspace: nothing to compute), as ``_plan_rope`` does."""
    problem = _cache_problem(key_cache, value_cache, key_scales, value_scales, query.dtype)
    b, h, n, d = key_cache.shape
    if query.dim() != 4 or query.shape[0] != b or query.shape[3] != d or h == 0 or query.shape[1] % h:
        raise ValueError(f"query must be ({b}, a multiple of {h}, M, {d}); got {tuple(query.shape)}.")
    if d == 0:
        raise ValueError("the head dimension must be positive.")
    hq, m = query.shape[1], query.shape[2]
    if m > 256:
        raise ValueError(f"{m} drafted tokens exceed 256.")
    _check_sizes(query_rows_per_cache_head=hq // h * m)
    if tree_mask is not None and (tree_mask.dtype != torch.bool or tuple(tree_mask.shape) not in ((m, m), (1, m, m), (b, m, m))):
        raise ValueError(f"tree_mask must be bool of shape ({m}, {m}) or ({b}, {m}, {m}); got {tree_mask.dtype} {tuple(tree_mask.shape)}.")
    given = (query, lengths, tree_mask)
    lengths = _lengths("lengths", lengths, b)
    scale = 1 / math.sqrt(d) if scale is None else scale
    if not abs(scale) <= 2.3e38:  # scale * log2(e) must be a finite fp32 number
        raise ValueError(f"scale must be a finite fp32 number of magnitude up to 2.3e38; got {scale}.")
    _check_devices(query.device, query=query, key_cache=key_cache, value_cache=value_cache, lengths=lengths,
                   tree_mask=tree_mask, key_scales=key_scales, value_scales=value_scales)
    if query.numel() == 0 or n == 0:
        return (problem, None, (b, hq, m, d), query.dtype, query.device, 0), query, lengths, tree_mask
    if query.stride(3) != 1 or query.data_ptr() % 16 or any(query.shape[i] > 1 and query.stride(i) % 8 for i in range(3)):
        query = query.clone(memory_format=torch.contiguous_format)  # the kernels copy queries 16 bytes at a time
    tree = nat.Tree(hq, m, (*query.stride()[:3], 1), _INDEX_BITS[lengths.dtype], (0, 0), scale)
    if tree_mask is not None:
        tree_mask = _rows(tree_mask)
        tree.mask_strides[:] = (tree_mask.stride(0) if tree_mask.dim() == 3 and tree_mask.shape[0] > 1 else 0, tree_mask.stride(-2))
    with _on_device(query.device.index):
        ws_bytes = nat.lib.fcr_tree_workspace_bytes(C.byref(problem), C.byref(tree), 0)
    if ws_bytes == 0:
        raise ValueError(nat.last_error())
    hit = (problem, tree, (b, hq, m, d), query.dtype, query.device, ws_bytes)
    if all(x is y for x, y in zip(given, (query, lengths, tree_mask))):
        _keep(_TREE_CACHE, signature, hit)
    return hit, query, lengths, tree_mask
