"""The work on which the serving operators are measured: norm and rotation of queries and keys, the quantised
KV cache, attention of drafted tokens over it.

``listed()`` are the fixed cases and ``draw(rng)`` makes further ones of the same ranges.  A case is a dict of plain
values.  ``prepare`` makes its inputs on the GPU, ``run`` makes one pass: the plain form (elementary torch operations in
32 bits, one rounding at the end), or the package's own operators when ``own`` is set.  ``exact`` gives the result from
the operator's definition in 64 bits and ``work`` counts what a pass cannot do without.
"""
import math

import torch

own = False

_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_CODES = {"fp8": torch.float8_e4m3fn, "int8": torch.int8}
_TOP = {"fp8": 448.0, "int8": 127.0}


# ----------------------------------------------------------------------------------------------------------- cases
def _rope(name, b, m, hq, hk, d, dtype="bf16", rotary=0, interleaved=False, norm=True, fused=True, far=0):
    """``rotary`` 0: the whole head is rotated.  ``fused``: q and k are views of one projection's (B, M, heads, D)
    output.  ``far``: the first position."""
    return {"name": name, "op": "rope", "b": b, "m": m, "hq": hq, "hk": hk, "d": d, "dtype": dtype,
            "rotary": rotary or d, "interleaved": interleaved, "norm": norm, "fused": fused, "far": far}


def _cache(name, b, h, cap, d, m, read, gather, fmt, dtype="bf16"):
    """Append ``m`` tokens per sequence to a cache of ``cap`` positions, then read ``read`` positions of every head:
    the first ones, or (``gather``) a selection of them in ascending order."""
    return {"name": name, "op": "cache", "b": b, "h": h, "cap": cap, "d": d, "m": m, "read": read, "gather": gather,
            "fmt": fmt, "dtype": dtype}


def _attn(name, b, hq, hk, n, m, d, fmt="none", dtype="bf16", mask="causal", ragged=True, shared_mask=False):
    """``m`` drafted tokens of each sequence over at most ``n`` cached ones.  ``mask``: "causal" (a chain), "tree"
    (random parents) or "sparse" (a tree with rows that attend no drafted token)."""
    return {"name": name, "op": "attn", "b": b, "hq": hq, "hk": hk, "n": n, "m": m, "d": d, "fmt": fmt,
            "dtype": dtype, "mask": mask, "ragged": ragged, "shared_mask": shared_mask}


def listed():
    return [
        # One decode step of one sequence: nothing but latency.
        _rope("rope_1x1", 1, 1, 32, 8, 128),
        # The drafted tokens of a serving batch, adjacent pairs rotated, fp16.
        _rope("rope_16x64_interleaved_fp16", 16, 64, 32, 8, 64, dtype="fp16", interleaved=True),
        # A chunk of a long prompt, far positions, as the fused projection leaves q and k.
        _rope("rope_2x16384_far", 2, 16384, 32, 8, 128, far=114688),
        # A token per sequence joins an int8 cache; the quarter of 8192 keys that a selection kept is read.
        _cache("cache_1_keep_2048_int8", 1, 32, 8192, 128, 1, 2048, True, "int8", dtype="fp16"),
        # A 509-token chunk of two prompts, then the 4096 keys so far for the next chunk.
        _cache("cache_509_read_4096_fp8", 2, 8, 4096, 80, 509, 4096, False, "fp8"),
        # Whole prompts are written and read back.
        _cache("cache_32768_fp8", 2, 8, 32768, 128, 32768, 32768, False, "fp8"),
        # One decode step over a short context in 16 bits: latency.
        _attn("token_1x4096", 1, 32, 8, 4096, 1, 128, ragged=False),
        # A decode step of a serving batch of ragged contexts over an fp8 cache.
        _attn("token_32x8191_fp8", 32, 32, 8, 8191, 1, 128, fmt="fp8"),
        # A long context, one sequence, fp16.
        _attn("token_1x131072_fp16", 1, 64, 8, 131072, 1, 128, dtype="fp16", ragged=False),
        # Trees of 26 drafted tokens, every head with its own keys, head dimension 80, one tree for the batch.
        _attn("tree_26_4x4096_d80_int8", 4, 20, 20, 4096, 26, 80, fmt="int8", dtype="fp16", mask="tree", shared_mask=True),
        # Trees of 16 drafted tokens in a serving batch over an int8 cache.
        _attn("tree_16_16x32768_int8", 16, 32, 8, 32768, 16, 128, fmt="int8", mask="sparse"),
        # Trees of 64 drafted tokens, 256 query rows per key head: the compute-bound end.
        _attn("tree_64_8x16384", 8, 32, 8, 16384, 64, 128, mask="tree"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["rope", "cache", "attn", "attn"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "rope":
        hk = rng.choice([1, 2, 4, 8, 16])
        hq = hk * rng.choice([1, 2, 4, 7, 8])
        d = rng.choice([64, 80, 96, 128, 128, 256])
        b = _log(rng, 1, 32)
        dtype = rng.choice([dtype, dtype, "fp32"])
        m = _log(rng, 1, max(1, min(16384, (2 * 16384 * 40 * 128) // (b * (hq + hk) * d * (2 if dtype == "fp32" else 1)))))
        c = _rope("", b, m, hq, hk, d, dtype=dtype, interleaved=rng.random() < 0.3,
                  rotary=rng.choice([0, 0, d // 2]), norm=rng.random() < 0.8, fused=rng.random() < 0.7,
                  far=rng.choice([0, 4095, 1000003]))
    elif op == "cache":
        h = rng.choice([1, 2, 4, 8, 20, 32])
        d = rng.choice([64, 80, 96, 128, 128])
        b = _log(rng, 1, 16)
        cap = _log(rng, 16, max(16, min(32768, (2 * 8 * 32768 * 128) // (b * h * d))))
        m = _log(rng, 1, cap)
        c = _cache("", b, h, cap, d, m, _log(rng, 1, cap), rng.random() < 0.5, rng.choice(["fp8", "int8"]), dtype=dtype)
    else:
        hk = rng.choice([1, 2, 4, 8, 20])
        g = rng.choice([1, 1, 2, 4, 7, 8])
        d = rng.choice([64, 80, 96, 128, 128])
        b = _log(rng, 1, 32)
        m = rng.choice([1, 1, 1, _log(rng, 2, 128), _log(rng, 2, 128)])
        fmt = rng.choice(["none", "fp8", "int8"])
        n = _log(rng, 1, max(1, min(131072, (8 * 32 * 10000 * 64) // (b * hk * g * m),
                                    (16 * 8 * (10000 if fmt == "none" else 20000) * 128) // (b * hk * d))))
        c = _attn("", b, hk * g, hk, n, m, d, fmt=fmt, dtype=dtype,
                  mask=rng.choice(["causal", "tree", "sparse"]) if m > 1 else "causal", ragged=rng.random() < 0.7,
                  shared_mask=rng.random() < 0.3)
    c.pop("name")
    return c


# ---------------------------------------------------------------------------------------------------------- inputs
def _unit(codes):
    """The values of codes in 32 bits."""
    return codes.float()


def _scale(scales):
    """The factors that a cache's scale bytes stand for: 2^(byte - 127), byte 255 is NaN."""
    bits = scales.view(torch.uint8)
    return torch.where(bits == 255, math.nan, torch.exp2(bits.float() - 127))


def _quantise(x, fmt):
    """Codes and scale bytes of the rows of x: the least power of two that brings a row's largest value to the
    format's, and the nearest codes, ties to even.  A row that holds a non-finite value becomes NaN."""
    largest = {torch.float16: 2.0 ** 15, torch.bfloat16: 2.0 ** 127}[x.dtype] * (1.875 if fmt == "fp8" else 1.96875)
    x = x.float()
    top = x.abs().amax(-1)
    fine = torch.isfinite(x).all(-1)
    mant, expo = torch.frexp(torch.where(fine, top, 0.0) / _TOP[fmt])  # exact enough: a border is met by exact quotients only
    e = torch.where(mant == 0.5, expo - 1, expo)
    e = torch.where(top == 0, -127, e).clamp(min=-127)
    y = torch.ldexp(torch.ldexp(x.clamp(-largest, largest), -(e // 2)[..., None]), -(e - e // 2)[..., None])
    y = torch.where(fine[..., None], y, 0.0)
    codes = y.to(torch.float8_e4m3fn) if fmt == "fp8" else torch.round(y).to(torch.int8)
    return codes, torch.where(fine, e + 127, 255).to(torch.uint8)


def _cached(b, h, cap, d, fmt, dtype, g, dev):
    """A cache tensor (b, h, cap, d) that holds earlier tokens, and its scales (None in 16 bits)."""
    if fmt == "none":
        x = torch.empty((b, h, cap, d), dtype=dtype, device=dev)
        for i in range(b):
            x[i] = torch.randn((h, cap, d), generator=g, device=dev)
        return x, None
    codes = torch.empty((b, h, cap, d), dtype=_CODES[fmt], device=dev)
    scales = torch.empty((b, h, cap), dtype=torch.uint8, device=dev)
    for i in range(b):
        # tokens differ in size, as keys do
        x = torch.randn((h, cap, d), generator=g, device=dev) * torch.exp(0.3 * torch.randn((h, cap, 1), generator=g, device=dev))
        codes[i], scales[i] = _quantise(x.to(dtype), fmt)
    return codes, scales.view(torch.float8_e8m0fnu)


def _tree(case, g, dev):
    """(B or 1, M, M) truth values: which drafted tokens each drafted token attends; None for a chain."""
    m = case["m"]
    if case["mask"] == "causal":
        return None
    b = 1 if case["shared_mask"] else case["b"]
    # a parent for each token among the ones before it; a token attends itself and its ancestors
    draw_ = torch.rand((b, m), generator=g, device=dev)
    parents = (draw_ * torch.arange(m, device=dev)).long()
    mask = torch.eye(m, dtype=torch.bool, device=dev).repeat(b, 1, 1)
    for i in range(1, m):
        mask[:, i] |= mask[torch.arange(b, device=dev), parents[:, i]]
    if case["mask"] == "sparse":  # slots that a short tree leaves empty
        mask &= torch.rand((b, m, 1), generator=g, device=dev) < 0.8
    return mask


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    t = _TYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] == "rope":
        b, m, hq, hk, d = (case[k] for k in ("b", "m", "hq", "hk", "d"))
        if case["fused"]:
            x = torch.randn((b, m, hq + hk, d), generator=g, device=dev).to(t).transpose(1, 2)
            s["q"], s["k"] = x[:, :hq], x[:, hq:]
        else:
            s["q"] = torch.randn((b, hq, m, d), generator=g, device=dev).to(t)
            s["k"] = torch.randn((b, hk, m, d), generator=g, device=dev).to(t)
        s["qw"] = s["kw"] = None
        if case["norm"]:
            s["qw"] = (1 + 0.1 * torch.randn((d,), generator=g, device=dev)).to(t)
            s["kw"] = (1 + 0.1 * torch.randn((d,), generator=g, device=dev)).to(t)
        r = case["rotary"]
        s["freq"] = (10000.0 ** (-torch.arange(0, r, 2, device=dev, dtype=torch.float64) / r)).float()
        start = torch.randint(0, 64, (b, 1), generator=g, device=dev) + case["far"]
        s["pos"] = (start + torch.arange(m, device=dev)).int()
    elif case["op"] == "cache":
        b, h, cap, d, m = (case[k] for k in ("b", "h", "cap", "d", "m"))
        s["kc"], s["ks"] = _cached(b, h, cap, d, case["fmt"], t, g, dev)
        s["vc"], s["vs"] = _cached(b, h, cap, d, case["fmt"], t, g, dev)
        x = torch.randn((b, m, 2 * h, d), generator=g, device=dev).to(t).transpose(1, 2)
        s["k"], s["v"] = x[:, :h], x[:, h:]
        s["lens"] = (torch.rand((b,), generator=g, device=dev) * (cap - m + 1)).int()
        s["sel"] = None
        if case["gather"]:
            keep = torch.rand((b, h, cap), generator=g, device=dev).topk(case["read"], dim=-1)[1]
            s["sel"] = keep.sort(-1)[0]
    else:
        b, hq, hk, n, m, d = (case[k] for k in ("b", "hq", "hk", "n", "m", "d"))
        s["q"] = torch.randn((b, m, hq, d), generator=g, device=dev).to(t).transpose(1, 2)
        s["kc"], s["ks"] = _cached(b, hk, n + m, d, case["fmt"], t, g, dev)
        s["vc"], s["vs"] = _cached(b, hk, n + m, d, case["fmt"], t, g, dev)
        s["lens"] = torch.full((b,), n, device=dev, dtype=torch.int32)
        if case["ragged"]:
            s["lens"] = (n * (0.25 + 0.75 * torch.rand((b,), generator=g, device=dev))).int()
        s["mask"] = _tree(case, g, dev)
    return s


# -------------------------------------------------------------------------------------------------------- one pass
def _plain_rotate(x, w, pos, freq, interleaved):
    y = x.float()
    if w is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * w.float()
    angle = pos.double()[:, None, :, None] * freq.double()
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    half = freq.numel()
    y, rest = y[..., : 2 * half], y[..., 2 * half :]
    if interleaved:
        a, c = y[..., 0::2], y[..., 1::2]
        y = torch.stack((a * cos - c * sin, a * sin + c * cos), -1).flatten(-2)
    else:
        a, c = y[..., :half], y[..., half:]
        y = torch.cat((a * cos - c * sin, a * sin + c * cos), -1)
    return torch.cat((y, rest), -1).to(x.dtype)


def _plain_append(x, fmt, codes, scales, lens):
    b, h, m, _ = x.shape
    new, bits = _quantise(x, fmt)
    at = (lens.long()[:, None] + torch.arange(m, device=x.device))[:, None, :].expand(b, h, m)
    codes.view(torch.uint8).scatter_(2, at[..., None].expand_as(new), new.view(torch.uint8))
    scales.view(torch.uint8).scatter_(2, at, bits)


def _plain_read(codes, scales, sel, n, dtype):
    raw, bits = codes.view(torch.uint8), scales.view(torch.uint8)
    if sel is None:
        raw, bits = raw[:, :, :n], bits[:, :, :n]
    else:
        raw, bits = raw.gather(2, sel[..., None].expand(*sel.shape, raw.shape[-1])), bits.gather(2, sel)
    return (_unit(raw.view(codes.dtype)) * _scale(bits)[..., None]).to(dtype)


def _plain_attention(s):
    c = s["case"]
    q = s["q"]
    b, hq, m, d = q.shape
    hk = c["hk"]
    k = _unit(s["kc"]) if s["ks"] is None else _unit(s["kc"]) * _scale(s["ks"])[..., None]
    v = _unit(s["vc"]) if s["vs"] is None else _unit(s["vc"]) * _scale(s["vs"])[..., None]
    n = k.shape[2]
    x = q.float().reshape(b, hk, (hq // hk) * m, d) @ k.transpose(-1, -2) * (1 / math.sqrt(d))
    x = x.view(b, hk, hq // hk, m, n)
    behind = torch.arange(n, device=q.device) - s["lens"][:, None]  # (B, n): a key's place among the drafted tokens
    drafted = s["mask"]
    if drafted is None:
        drafted = torch.ones((1, m, m), dtype=torch.bool, device=q.device).tril()
    at = behind.clamp(0, m - 1)[:, None, :].expand(b, m, n)
    seen = drafted.expand(b, m, m).gather(2, at) & ((behind >= 0) & (behind < m))[:, None]
    seen = (seen | (behind < 0)[:, None])[:, None, None]
    x = x.masked_fill(~seen, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = (p.view(b, hk, -1, n) @ v).view(b, hk, hq // hk, m, d) / torch.where(total == 0, 1.0, total)
    lse = (torch.where(total == 0, -math.inf, torch.log(total)) + torch.where(top == -math.inf, 0.0, top)).squeeze(-1)
    return out.view(b, hq, m, d).to(q.dtype), lse.view(b, hq, m)


def run(state):
    s = state
    c = s["case"]
    if own:
        import flash_colreduce_b200 as fcr

        if c["op"] == "rope":
            return fcr.qk_norm_rope(s["q"], s["k"], s["pos"], s["freq"], s["qw"], s["kw"], eps=1e-6, interleaved=c["interleaved"])
        if c["op"] == "cache":
            fcr.kv_cache_append(s["k"], s["v"], s["kc"], s["vc"], s["lens"], s["ks"], s["vs"])
            return fcr.kv_cache_read(s["kc"], s["vc"], s["ks"], s["vs"], positions=s["sel"],
                                     n=None if c["gather"] else c["read"], dtype=s["k"].dtype)
        return fcr.tree_attention(s["q"], s["kc"], s["vc"], s["lens"], s["mask"], key_scales=s["ks"], value_scales=s["vs"],
                                  return_lse=True)
    if c["op"] == "rope":
        return (_plain_rotate(s["q"], s["qw"], s["pos"], s["freq"], c["interleaved"]),
                _plain_rotate(s["k"], s["kw"], s["pos"], s["freq"], c["interleaved"]))
    if c["op"] == "cache":
        _plain_append(s["k"], c["fmt"], s["kc"], s["ks"], s["lens"])
        _plain_append(s["v"], c["fmt"], s["vc"], s["vs"], s["lens"])
        return (_plain_read(s["kc"], s["ks"], s["sel"], c["read"], s["k"].dtype),
                _plain_read(s["vc"], s["vs"], s["sel"], c["read"], s["k"].dtype))
    return _plain_attention(s)


# ---------------------------------------------------------------------------------------------- 64 bits and amounts
def _exact_rotate(x, w, pos, freq, interleaved):
    y = x.double()
    if w is not None:
        y = y / (y.pow(2).sum(-1, keepdim=True) / y.shape[-1] + 1e-6).sqrt() * w.double()
    out = y.clone()
    half = freq.numel()
    first = torch.arange(half, device=x.device) * (2 if interleaved else 1)
    second = first + (1 if interleaved else half)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=x.device), torch.einsum("bm,i->bmi", pos.double(), freq.double()))[:, None]
    z = torch.complex(y[..., first], y[..., second]) * turn
    out[..., first], out[..., second] = z.real, z.imag
    return out


def _exact_written(x, fmt):
    """The values that a cache stands for after rows x are written, in 64 bits."""
    y = x.double()
    top = y.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(top / _TOP[fmt]))
    for step in (-1, 1):  # a logarithm next to a whole number: the least e with top <= largest * 2^e
        e = torch.where((top <= _TOP[fmt] * torch.exp2(e + step)) if step < 0 else (top > _TOP[fmt] * torch.exp2(e)), e + step, e)
    u = y / torch.exp2(e)
    if fmt == "int8":
        return torch.round(u) * torch.exp2(e)
    size = torch.floor(torch.log2(u.abs().clamp(min=2.0 ** -6)))  # below 2^-6 the codes are evenly spaced
    grid = torch.exp2(size - 3)
    return torch.round(u / grid) * grid * torch.exp2(e)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        return (_exact_rotate(s["q"], s["qw"], s["pos"], s["freq"], case["interleaved"]),
                _exact_rotate(s["k"], s["kw"], s["pos"], s["freq"], case["interleaved"]))

    def values(codes, scales):
        return codes.double() if scales is None else codes.double() * torch.exp2(scales.view(torch.uint8).double() - 127)[..., None]

    if case["op"] == "cache":
        found = []
        for x, codes, scales in ((s["k"], s["kc"], s["ks"]), (s["v"], s["vc"], s["vs"])):
            now = values(codes, scales)
            for i in range(case["b"]):
                at = int(s["lens"][i])
                now[i, :, at : at + case["m"]] = _exact_written(x[i], case["fmt"])
            if s["sel"] is None:
                found.append(now[:, :, : case["read"]])
            else:
                found.append(torch.take_along_dim(now, s["sel"][..., None], 2))
        return tuple(found)
    b, hq, hk, m, d = (case[k] for k in ("b", "hq", "hk", "m", "d"))
    out = torch.zeros((b, hq, m, d), dtype=torch.float64, device=s["q"].device)
    lse = torch.full((b, hq, m), -math.inf, dtype=torch.float64, device=s["q"].device)
    for i in range(b):
        have = int(s["lens"][i])
        chain = torch.ones((m, m), dtype=torch.bool, device=s["q"].device).tril()
        mask = chain if s["mask"] is None else s["mask"][0 if case["shared_mask"] else i]
        seen = torch.cat((torch.ones((m, have), dtype=torch.bool, device=mask.device), mask), 1)
        bias = torch.zeros(seen.shape, dtype=torch.float64, device=mask.device).masked_fill(~seen, -math.inf)
        empty = ~seen.any(1)
        k = values(s["kc"][i], None if s["ks"] is None else s["ks"][i])[:, : have + m]
        v = values(s["vc"][i], None if s["vs"] is None else s["vs"][i])[:, : have + m]
        for h in range(hq):
            x = s["q"][i, h].double() @ k[h // (hq // hk)].T / d ** 0.5 + bias
            w = torch.softmax(x, -1).masked_fill(empty[:, None], 0.0)
            out[i, h], lse[i, h] = w @ v[h // (hq // hk)], torch.logsumexp(x, -1)
    return out, lse


def work(case):
    size = {"fp16": 2, "bf16": 2, "fp32": 4}[case["dtype"]]
    if case["op"] == "rope":
        values = case["b"] * case["m"] * (case["hq"] + case["hk"]) * case["d"]
        return {"bytes": 2 * values * size + case["b"] * case["m"] * 4, "flops": 8 * values}
    if case["op"] == "cache":
        new = 2 * case["b"] * case["h"] * case["m"]  # rows of keys and of values
        read = 2 * case["b"] * case["h"] * case["read"]
        d = case["d"]
        return {"bytes": new * (d * size + d + 1) + read * (d * size + d + 1) + (read * 4 if case["gather"] else 0),
                "flops": 3 * new * d + read * d}
    share = 0.625 if case["ragged"] else 1.0  # the mean of the drawn lengths
    keys = int(case["n"] * share) + case["m"]
    row = case["d"] * size if case["fmt"] == "none" else case["d"] + 1
    queries = case["b"] * case["hq"] * case["m"]
    return {"bytes": 2 * case["b"] * case["hk"] * keys * row + 2 * queries * case["d"] * size + 4 * queries,
            "flops": 4 * queries * keys * case["d"]}
