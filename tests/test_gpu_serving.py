"""The serving operators against their definitions in 64 bits (needs a B200).

Tolerances.  u = finfo.eps / 2 is the relative error of one rounding to the output's type.

rope: one rounding of the result (u * |y|) on top of the fp32 arithmetic.  With e = 2^-24 that is at most: 13 additions of the
squares, halved by the root, 1 for the mean, 2 for rsqrtf and 2 products (12 e), 4 e for a cosine or sine of 2 ulp, 3.2 e for
the fraction of a turn rounded to fp32 (pi * e of angle), 3 e for the two products and the sum: under 32 e of |a| + |b|.

cache: codes and scales are equal, reading is exact.

attention: a weight p has the relative error of its score's absolute one -- the 32-bit dot product, at most
(D / 16 + 4) * 2^-22 of scale * sum |q||k| -- plus 2^-21 for the exponential and its argument's rounding (2^-23 of the largest
score), and is rounded to 16 bits once (u): together `pe`.  Numerator and denominator both carry it, so out is off by at most
2 * pe * sum p|v| / sum p, plus u * |out| for its own rounding.  lse is off by the scores' and exponentials' part alone.
"""
import math

import pytest
import torch

import flash_colreduce_b200 as fc
from oracle.serving_oracle import attention, dequantize_rows, quantize_rows, rope

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
FP8, I8 = torch.float8_e4m3fn, torch.int8
DEV = "cuda:0"


def _u(dtype):
    return torch.finfo(dtype).eps / 2


# ------------------------------------------------------------------------------------------------------------- rope
def _rope_inputs(b, hq, hk, m, d, dtype, seed=0, weight_dtype=None):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(b, hq, m, d, generator=g).to(dtype)
    k = torch.randn(b, hk, m, d, generator=g).to(dtype)
    qw = (1 + 0.2 * torch.randn(d, generator=g)).to(weight_dtype or dtype)
    kw = (1 + 0.2 * torch.randn(d, generator=g)).to(weight_dtype or dtype)
    return q, k, qw, kw


def _freq(r, base=10000.0):
    return (base ** (-torch.arange(0, r, 2, dtype=torch.float64) / r)).float()


def _check_rope(got, x, pos, freq, w, interleaved, eps=1e-6):
    want = rope(x, pos, freq, w, eps, interleaved)
    y = x.double()
    if w is not None:
        y = y / torch.sqrt(y.pow(2).mean(-1, keepdim=True) + eps) * w.double()
    size = y.abs()
    half = freq.numel()
    first = slice(0, 2 * half, 2) if interleaved else slice(0, half)
    second = slice(1, 2 * half, 2) if interleaved else slice(half, 2 * half)
    pair = size[..., first] + size[..., second]
    size[..., first], size[..., second] = pair, pair
    tiny = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    bound = _u(x.dtype) * want.abs() + 32 * 2.0 ** -24 * size + tiny
    assert got.shape == x.shape and got.dtype == x.dtype and got.is_contiguous()
    worst = ((got.cpu().double() - want).abs() / bound).max().item()
    assert worst <= 1.0, worst


@pytest.mark.parametrize("dtype", [BF, HF, torch.float32])
@pytest.mark.parametrize("b,hq,hk,m,d,rotary,interleaved", [
    (1, 32, 8, 1, 128, 128, False), (1, 32, 8, 1, 128, 128, True), (2, 4, 4, 37, 64, 64, False), (2, 4, 2, 37, 64, 64, True),
    (3, 7, 1, 129, 256, 256, False), (1, 2, 1, 5, 256, 256, True), (2, 20, 20, 9, 80, 80, False), (2, 3, 2, 9, 96, 48, True),
    (1, 1, 1, 1, 2, 2, False), (1, 5, 3, 11, 33, 20, False), (1, 2, 2, 3, 128, 0, False), (1, 2, 2, 3, 128, 64, False),
    (1, 40, 8, 700, 128, 128, False), (2, 8, 0, 3, 64, 64, False), (2, 0, 8, 3, 64, 64, False),
])
def test_rope(dtype, b, hq, hk, m, d, rotary, interleaved):
    q, k, qw, kw = _rope_inputs(b, hq, hk, m, d, dtype, seed=m + d)
    freq = _freq(rotary) if rotary else torch.zeros(0)
    pos = torch.randint(0, 5000, (b, m), generator=torch.Generator().manual_seed(1), dtype=torch.int32)
    got_q, got_k = fc.qk_norm_rope(q.to(DEV), k.to(DEV), pos.to(DEV), freq.to(DEV), qw.to(DEV), kw.to(DEV), interleaved=interleaved)
    if hq:
        _check_rope(got_q, q, pos, freq, qw, interleaved)
    if hk:
        _check_rope(got_k, k, pos, freq, kw, interleaved)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("weights", ["none", "q", "fp32"])
def test_rope_without_weights_and_with_fp32_ones(dtype, weights):
    q, k, qw, kw = _rope_inputs(2, 6, 2, 19, 128, dtype, weight_dtype=torch.float32 if weights == "fp32" else None)
    pos = torch.arange(100, 119)  # int64, shared by the batch
    freq = _freq(128)
    a, c = (None, None) if weights == "none" else (qw, None) if weights == "q" else (qw, kw)
    got_q, got_k = fc.qk_norm_rope(q.to(DEV), k.to(DEV), pos.to(DEV), freq.to(DEV), None if a is None else a.to(DEV),
                                   None if c is None else c.to(DEV), eps=1e-5)
    _check_rope(got_q, q, pos, freq, a, False, 1e-5)
    _check_rope(got_k, k, pos, freq, c, False, 1e-5)


@pytest.mark.parametrize("d", [64, 80, 128])
def test_rope_far_and_negative_positions(d):
    q, k, qw, kw = _rope_inputs(1, 4, 2, 6, d, torch.float32)
    pos = torch.tensor([0, 1, 1000003, 2 ** 31 - 1, 2 ** 40 + 12345, -7])
    freq = _freq(d)
    got_q, got_k = fc.qk_norm_rope(q.to(DEV), k.to(DEV), pos.to(DEV), freq.to(DEV), qw.to(DEV), kw.to(DEV))
    # 2^40 positions are 2^37.4 turns: 2^-53 of them is 3e-5 of a turn, 1.9e-4 of angle; the others are far below one rounding
    keep = [0, 1, 2, 3, 5]
    _check_rope(got_q[:, :, keep].contiguous(), q[:, :, keep], pos[keep], freq, qw, False)
    _check_rope(got_k[:, :, keep].contiguous(), k[:, :, keep], pos[keep], freq, kw, False)
    want = rope(q[:, :, 4:5], pos[4:5], freq, qw)
    assert (got_q[:, :, 4:5].cpu().double() - want).abs().max() < 2e-3


@pytest.mark.parametrize("d", [64, 80, 128])
def test_rope_of_views(d):
    """A fused projection's output, an odd offset, a reversed batch, an innermost stride that is not 1."""
    g = torch.Generator().manual_seed(4)
    x = torch.randn(2, 13, 12 * d + 1, generator=g).to(BF).to(DEV)
    pos, freq = torch.arange(13, device=DEV, dtype=torch.int32), _freq(d).to(DEV)
    w = torch.ones(d, dtype=BF, device=DEV)
    for off in (0, 1):
        v = x[..., off : off + 12 * d].view(2, 13, 12, d).transpose(1, 2)
        got_q, got_k = fc.qk_norm_rope(v[:, :8], v[:, 8:10], pos, freq, w, w)
        _check_rope(got_q, v[:, :8].cpu(), pos.cpu(), freq.cpu(), w.cpu(), False)
        _check_rope(got_k, v[:, 8:10].cpu(), pos.cpu(), freq.cpu(), w.cpu(), False)
    t = torch.randn(2, 4, d, 13, generator=g).to(BF).to(DEV).transpose(2, 3)
    got_q, _ = fc.qk_norm_rope(t, t, pos, freq, w, w)
    _check_rope(got_q, t.cpu(), pos.cpu(), freq.cpu(), w.cpu(), False)


def test_rope_non_finite_values_stay_in_their_rows():
    q, k, qw, kw = _rope_inputs(1, 4, 2, 6, 128, BF)
    pos, freq = torch.arange(6), _freq(128)
    args = [x.to(DEV) for x in (pos, freq, qw, kw)]
    clean, _ = fc.qk_norm_rope(q.to(DEV), k.to(DEV), *args)
    q[0, 1, 2, 5], q[0, 3, 4, 0] = float("nan"), float("inf")
    got, _ = fc.qk_norm_rope(q.to(DEV), k.to(DEV), *args)
    bad = torch.zeros(1, 4, 6, dtype=torch.bool, device=DEV)
    bad[0, 1, 2] = bad[0, 3, 4] = True
    assert torch.equal(got[~bad], clean[~bad]) and got[0, 1, 2].isnan().any() and got[0, 3, 4].isnan().any()


# ------------------------------------------------------------------------------------------------------------ cache
def _empty_cache(b, h, n, d, fmt, fill=0x5a):
    kind = {BF: torch.int16, HF: torch.int16}.get(fmt, torch.uint8)
    data = [torch.full((b, h, n, d), fill, dtype=kind, device=DEV).view(fmt) for _ in range(2)]
    if fmt in (BF, HF):
        return (*data, None, None)
    return (*data, *[torch.full((b, h, n), fill, dtype=torch.uint8, device=DEV).view(torch.float8_e8m0fnu) for _ in range(2)])


def _bits(x):
    return x.view(torch.int16 if x.dtype in (BF, HF) else torch.uint8).cpu()


def _expected_write(x, cache, scales, lens, counts, fmt):
    """The cache's bits after the write, from the definition."""
    want, ws = _bits(cache).clone(), None if scales is None else _bits(scales).clone()
    codes, bits = (None, None) if scales is None else quantize_rows(x, fmt)
    for b in range(x.shape[0]):
        for m in range(x.shape[2]):
            at = int(lens[b]) + m
            if int(lens[b]) < 0 or at >= want.shape[2] or (counts is not None and m >= int(counts[b])):
                continue
            if scales is None:
                want[b, :, at] = x[b, :, m].view(torch.int16)
            else:
                want[b, :, at] = codes[b, :, m].to(fmt).view(torch.uint8)
                ws[b, :, at] = bits[b, :, m]
    return want, ws


def _same_codes(got, want, fmt):
    if fmt == FP8:  # a negative value that rounds to zero is -0
        return torch.equal(got.view(FP8).float(), want.view(FP8).float())
    return torch.equal(got, want)


@pytest.mark.parametrize("fmt", ["16", FP8, I8])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("b,h,n,d,m,lens,counts", [
    (1, 1, 1, 8, 1, [0], None), (2, 3, 40, 128, 7, [0, 33], None), (2, 2, 40, 80, 9, [35, 2], [9, 3]), (3, 1, 9, 64, 4, [9, -1, 6], None),
    (2, 2, 20, 33, 5, [1, 18], [0, 5]), (1, 20, 300, 96, 257, [11], None), (2, 2, 16, 256, 3, [4, 13], None), (1, 1, 5, 1, 2, [1], None),
    (2, 1, 30, 128, 3, [0, 2 ** 31 - 1], None),
])
def test_append_and_read(fmt, dtype, b, h, n, d, m, lens, counts):
    fmt = dtype if fmt == "16" else fmt
    g = torch.Generator().manual_seed(n + d)
    x = (torch.randn(2, b, h, m, d, generator=g) * torch.exp(2 * torch.randn(2, b, h, m, 1, generator=g))).to(dtype)
    cache = _empty_cache(b, h, n, d, fmt)
    want = [_expected_write(x[i], cache[i], cache[2 + i], lens, counts, fmt) for i in range(2)]
    itype = torch.int32 if d != 96 else torch.int64
    fc.kv_cache_append(x[0].to(DEV), x[1].to(DEV), cache[0], cache[1], torch.tensor(lens, dtype=itype, device=DEV), cache[2], cache[3],
                       None if counts is None else torch.tensor(counts, dtype=itype, device=DEV))
    for i in range(2):
        assert _same_codes(_bits(cache[i]), want[i][0], fmt)
        if cache[2] is not None:
            assert torch.equal(_bits(cache[2 + i]), want[i][1])
    got = fc.kv_cache_read(*cache, dtype=dtype)
    for i in range(2):
        if cache[2] is None:
            assert torch.equal(_bits(got[i]), want[i][0])
        else:
            assert torch.equal(got[i].cpu().double(), dequantize_rows(want[i][0].view(fmt), want[i][1]).to(dtype).double())
    # a part, and a selection with positions that do not exist
    part = fc.kv_cache_read(*cache, n=n // 2, dtype=dtype)
    assert torch.equal(part[1], got[1][:, :, : n // 2])
    for ptype in (torch.int32, torch.int64):
        sel = torch.randint(0, n, (b, h, 2 * n + 1), generator=g).to(ptype).to(DEV)
        sel[..., 0], sel[..., -1] = -1, n
        picked = fc.kv_cache_read(*cache, positions=sel, dtype=dtype)
        at = sel[..., 1:-1].long()[..., None].expand(b, h, 2 * n - 1, d)
        for i in range(2):
            assert torch.equal(picked[i][:, :, 1:-1], got[i].gather(2, at))
            assert (picked[i][:, :, 0] == 0).all() and (picked[i][:, :, -1] == 0).all()


@pytest.mark.parametrize("fmt", [FP8, I8])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_written_rows_at_the_ends_of_the_range(fmt, dtype):
    fi = torch.finfo(dtype)
    tiny = fi.smallest_normal * fi.eps
    rows = [[0.0] * 16, [fi.max, -fi.max] * 8, [tiny, -tiny] * 8, [1.0] * 15 + [float("nan")], [float("-inf")] + [2.0] * 15,
            [0.5 * fi.max, 448.0, 127.0, 1.0] * 4, [448.0] * 16, [127.0] * 16, [449.0] * 16, [127.5, 63.5, 0.5, 1.5] * 4, [-0.0] * 16,
            [224.0, 17.0, 18.0, 19.0] * 4, [fi.smallest_normal, tiny, 0.0, -tiny] * 4]
    x = torch.tensor(rows, dtype=torch.float64).to(dtype).view(1, 1, len(rows), 16)
    cache = _empty_cache(1, 1, len(rows), 16, fmt)
    want, ws = _expected_write(x, cache[0], cache[2], [0], None, fmt)
    fc.kv_cache_append(x.to(DEV), x.to(DEV), cache[0], cache[1], torch.zeros(1, dtype=torch.int32, device=DEV), cache[2], cache[3])
    assert _same_codes(_bits(cache[0]), want, fmt) and torch.equal(_bits(cache[2]), ws)
    got, _ = fc.kv_cache_read(*cache, dtype=dtype)
    exact = dequantize_rows(want.view(fmt), ws)
    assert torch.equal(got.cpu().double().nan_to_num(7.0), exact.nan_to_num(7.0))
    assert torch.equal(got.isnan().all(-1).flatten().cpu(), (ws == 255).flatten())


@pytest.mark.parametrize("fmt", [FP8, I8, BF])
def test_append_and_read_of_views(fmt):
    """A fused projection's output into a slice of a larger cache, at aligned and odd offsets; what lies around it stays."""
    g = torch.Generator().manual_seed(8)
    big = _empty_cache(3, 4, 50, 96, fmt)
    for off in (0, 1):
        x = torch.randn(2, 6, 4 * 64 + 1, generator=g).to(BF).to(DEV)[..., off : off + 256].view(2, 6, 4, 64).transpose(1, 2)
        view = [None if c is None else c[1:, ::2, 5:45] for c in big]
        view[0], view[1] = view[0][..., 16 - off : 80 - off], view[1][..., 16 - off : 80 - off]
        before = [None if c is None else _bits(c).clone() for c in big]
        lens = [3, 36]
        want = [_expected_write(x[:, 2 * i : 2 * i + 2].cpu().contiguous(), view[i], view[2 + i], lens, None, fmt) for i in range(2)]
        fc.kv_cache_append(x[:, :2], x[:, 2:], view[0], view[1], torch.tensor(lens, device=DEV), view[2], view[3])
        for i in range(2):
            assert _same_codes(_bits(view[i].contiguous()), want[i][0], fmt)
            outside = _bits(big[i]).clone()
            outside[1:, ::2, 5:45, 16 - off : 80 - off] = before[i][1:, ::2, 5:45, 16 - off : 80 - off]
            assert torch.equal(outside, before[i])
        got = fc.kv_cache_read(*view, dtype=BF)
        for i in range(2):
            exact = want[i][0].view(BF) if view[2] is None else dequantize_rows(want[i][0].view(fmt), want[i][1]).to(BF)
            assert torch.equal(got[i].cpu(), exact)


# -------------------------------------------------------------------------------------------------------- attention
def _make(b, hq, h, m, n, d, fmt, dtype, seed=0):
    """Queries, a full cache of n positions and the values it stands for."""
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(b, hq, m, d, generator=g).to(dtype)
    x = (torch.randn(2, b, h, n, d, generator=g) * torch.exp(0.3 * torch.randn(2, b, h, n, 1, generator=g))).to(dtype)
    if fmt == "16":
        return q, [x[0].to(DEV), x[1].to(DEV), None, None], x.double()
    cache, values = [None] * 4, []
    for i in range(2):
        codes, bits = quantize_rows(x[i], fmt)
        cache[i], cache[2 + i] = codes.to(fmt).to(DEV), bits.to(DEV).view(torch.float8_e8m0fnu)
        values.append(dequantize_rows(codes, bits))
    return q, cache, torch.stack(values)


def _check_attention(got, lse, q, k, v, lens, mask, scale=None):
    b, hq, m, d = q.shape
    want, want_lse, weight = attention(q, k, v, lens, mask, scale)
    s = abs(1 / math.sqrt(d) if scale is None else scale)
    finite = lambda x: torch.where(torch.isfinite(x), x, 0.0).abs()  # noqa: E731
    big = s * (finite(q.double()).reshape(b, k.shape[1], -1, d) @ finite(k).transpose(-1, -2)).amax().item()  # largest sum |q||k| * scale
    score = big * (d / 16 + 4) * 2.0 ** -22 + big * 2.0 ** -23 + 2.0 ** -21
    u = _u(q.dtype)
    tiny = torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps
    bound = u * want.abs() + 2 * (u + score) * weight + tiny
    assert got.shape == q.shape and got.dtype == q.dtype
    gd = got.cpu().double()
    same_nan = torch.equal(gd.isnan(), want.isnan())
    assert same_nan, "NaN in other places"
    ok = torch.isfinite(want)
    worst = ((gd - want)[ok].abs() / bound[ok]).max().item() if ok.any() else 0.0
    assert worst <= 1.0, worst
    if lse is not None:
        gl = lse.cpu().double()
        empty = torch.isinf(want_lse) & (want_lse < 0)
        assert torch.equal(torch.isinf(gl) & (gl < 0), empty) and torch.equal(gl.isnan(), want_lse.isnan())
        fine = torch.isfinite(want_lse)
        if fine.any():
            assert ((gl - want_lse)[fine].abs() <= score + 2.0 ** -22 * want_lse[fine].abs() + 2.0 ** -20).all()


def _tree(b, m, seed, keep=1.0):
    g = torch.Generator().manual_seed(seed)
    mask = torch.eye(m, dtype=torch.bool).repeat(b, 1, 1)
    for x in range(b):
        for i in range(1, m):
            mask[x, i] |= mask[x, int(torch.randint(0, i, (1,), generator=g))]
    return mask & (torch.rand(b, m, 1, generator=g) < keep)


def _run(q, cache, lens, mask=None, scale=None, itype=torch.int32):
    return fc.tree_attention(q.to(DEV), cache[0], cache[1], torch.tensor(lens, dtype=itype, device=DEV),
                             None if mask is None else mask.to(DEV), scale, cache[2], cache[3], return_lse=True)


@pytest.mark.parametrize("fmt", ["16", FP8, I8])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("b,hq,h,m,n,d,lens", [
    (1, 1, 1, 1, 1, 16, [0]), (1, 8, 2, 1, 700, 128, [699]), (3, 8, 1, 1, 400, 128, [0, 1, 399]), (5, 4, 4, 1, 300, 64, [126, 127, 128, 129, 254]),
    (2, 6, 2, 5, 530, 80, [517, 3]), (2, 4, 1, 9, 260, 96, [0, 251]), (1, 8, 1, 8, 1300, 128, [1290]), (2, 8, 2, 16, 640, 64, [600, 129]),
    (2, 7, 1, 16, 333, 128, [317, 40]), (1, 20, 20, 26, 282, 80, [256]), (1, 8, 1, 31, 500, 128, [400]), (1, 8, 1, 64, 650, 128, [500]),
    (1, 9, 1, 64, 400, 64, [300]), (1, 2, 1, 256, 600, 128, [344]), (2, 2, 2, 128, 300, 32, [100, 172]), (1, 16, 16, 3, 5000, 128, [4997]),
    (4, 2, 1, 2, 200, 48, [10, 199, 198, 0]),
])
def test_attention_of_a_chain(fmt, dtype, b, hq, h, m, n, d, lens):
    q, cache, x = _make(b, hq, h, m, n, d, fmt, dtype, seed=m + n)
    got, lse = _run(q, cache, lens, itype=torch.int64 if m == 1 else torch.int32)
    _check_attention(got, lse, q, x[0], x[1], lens, None)
    again, lse2 = _run(q, cache, lens)
    assert torch.equal(got, again) and torch.equal(lse, lse2)
    alone = fc.tree_attention(q.to(DEV), cache[0], cache[1], torch.tensor(lens, device=DEV), key_scales=cache[2], value_scales=cache[3])
    assert torch.equal(got, alone)


@pytest.mark.parametrize("fmt", ["16", FP8, I8])
@pytest.mark.parametrize("b,hq,h,m,n,d,lens,shared", [
    (2, 4, 2, 7, 300, 128, [293, 0], False), (2, 8, 1, 16, 300, 64, [250, 120], True), (1, 4, 1, 33, 400, 128, [367], False),
    (2, 8, 2, 64, 800, 128, [700, 64], False), (1, 3, 1, 100, 300, 80, [128], True), (1, 2, 2, 256, 512, 64, [250], False),
    (3, 2, 1, 63, 200, 128, [0, 1, 127], False),
])
def test_attention_of_a_tree(fmt, b, hq, h, m, n, d, lens, shared):
    dtype = HF if m % 2 else BF
    q, cache, x = _make(b, hq, h, m, n, d, fmt, dtype, seed=n)
    mask = _tree(1 if shared else b, m, seed=m, keep=0.8)
    if shared:
        mask = mask[0]
    got, lse = _run(q, cache, lens, mask)
    _check_attention(got, lse, q, x[0], x[1], lens, mask)


@pytest.mark.parametrize("fmt", ["16", FP8, I8])
@pytest.mark.parametrize("m,g", [(1, 4), (6, 4), (16, 8), (40, 8)])
def test_rows_that_attend_nothing(fmt, m, g):
    q, cache, x = _make(3, g, 1, m, 150, 64, fmt, BF)
    mask = torch.zeros(m, m, dtype=torch.bool)
    got, lse = _run(q, cache, [0, 100, -5], mask)
    assert (got[0] == 0).all() and (got[2] == 0).all() and (lse[0] == -math.inf).all() and (lse[2] == -math.inf).all()
    _check_attention(got, lse, q, x[0], x[1], [0, 100, 0], mask)


@pytest.mark.parametrize("fmt", ["16", FP8, I8])
@pytest.mark.parametrize("m,g,d", [(1, 4, 128), (5, 4, 128), (24, 8, 64), (64, 8, 128)])
def test_masked_and_unwritten_positions_do_not_matter(fmt, m, g, d):
    n, lens = 420, [200, 131]
    q, cache, x = _make(2, g, 1, m, n, d, fmt, BF, seed=5)
    mask = _tree(2, m, seed=3)
    if m > 4:
        mask[:, :, 3] = False  # no token attends the fourth drafted one
    clean, clean_lse = _run(q, cache, lens, mask)
    for i in range(2):
        for b, at in enumerate(lens):
            if fmt == "16":
                cache[i][b, :, at + m :] = float("nan")
                if m > 4:
                    cache[i][b, :, at + 3] = float("inf")
            else:
                bits, codes = cache[2 + i].view(torch.uint8), cache[i].view(torch.uint8)
                bits[b, :, at + m :] = 255
                codes[b, :, at + m + 2 :] = 0x7f
                if m > 4:
                    bits[b, :, at + 3] = 255
    got, lse = _run(q, cache, lens, mask)
    assert torch.equal(got, clean) and torch.equal(lse, clean_lse)


@pytest.mark.parametrize("fmt", ["16", FP8])
@pytest.mark.parametrize("m,g,d", [(5, 4, 128), (24, 8, 64), (64, 8, 128)])
def test_a_non_finite_drafted_value_reaches_the_rows_that_attend_it_only(fmt, m, g, d):
    lens = [200]
    q, cache, x = _make(1, g, 1, m, 300, d, fmt, HF, seed=6)
    mask = _tree(1, m, seed=4)
    mask[0, : m // 2, 2] = False
    mask[0, m // 2 :, 2] = True
    if fmt == "16":
        cache[1][0, 0, 202, 3] = float("nan")
        cache[1][0, 0, 202, 7] = float("-inf")
        x[1][0, 0, 202, 3], x[1][0, 0, 202, 7] = float("nan"), float("-inf")
    else:
        cache[3].view(torch.uint8)[0, 0, 202] = 255
        x[1][0, 0, 202] = float("nan")
    got, lse = _run(q, cache, lens, mask)
    _check_attention(got, lse, q, x[0], x[1], lens, mask)
    if fmt == "16":
        assert (got[0, :, m // 2 :, 7] == -math.inf).all()


@pytest.mark.parametrize("fmt", ["16", I8])
@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0, 30.0])
def test_attention_scales(fmt, scale):
    q, cache, x = _make(1, 4, 2, 6, 300, 64, fmt, HF)
    got, lse = _run(q, cache, [290], scale=scale)
    _check_attention(got, lse, q, x[0], x[1], [290], None, scale)


@pytest.mark.parametrize("m", [1, 20])
def test_scores_that_grow_along_the_keys(m):
    """The running maximum rises in every tile, and falls from the first on."""
    g = torch.Generator().manual_seed(1)
    n, d = 1500, 64
    for ramp in (torch.linspace(0, 40, n), torch.linspace(40, 0, n)):
        q = torch.ones(1, 4, m, d).to(HF)
        k = (ramp[:, None] / 8 * torch.ones(n, d) + 0.01 * torch.randn(n, d, generator=g)).to(HF).view(1, 1, n, d)
        v = torch.randn(1, 1, n, d, generator=g).to(HF)
        got, lse = _run(q, [k.to(DEV), v.to(DEV), None, None], [n - m])
        _check_attention(got, lse, q, k.double(), v.double(), [n - m], None)


def test_cache_views_and_query_views():
    """A (B, M, Hq, D) projection's queries, an innermost stride other than 1, a slice of a larger cache, a mask's slice."""
    g = torch.Generator().manual_seed(9)
    b, hq, h, m, d = 2, 6, 2, 10, 64
    big = torch.randn(2, 3, 400, 2 * h, d + 32, generator=g).to(BF).to(DEV)  # (.., B, N, heads, D)
    k, v = (big[i, 1:, 30:360, h:, 16 : 16 + d].transpose(1, 2) for i in range(2))
    q = torch.randn(b, m, hq, d + 1, generator=g).to(BF).to(DEV)[..., 1:].transpose(1, 2)
    mask = torch.zeros(b, m + 3, m + 5, dtype=torch.bool)
    mask[:, 1 : m + 1, 2 : m + 2] = _tree(b, m, seed=2)
    lens = torch.tensor([320, 77], device=DEV)
    part = mask.to(DEV)[:, 1 : m + 1, 2 : m + 2]
    got, lse = fc.tree_attention(q, k, v, lens, part, return_lse=True)
    _check_attention(got, lse, q.cpu(), k.cpu().double(), v.cpu().double(), [320, 77], part.cpu())
    turned = part.transpose(1, 2).contiguous().transpose(1, 2)
    got2 = fc.tree_attention(q.transpose(2, 3).contiguous().transpose(2, 3), k, v, lens, turned)
    assert torch.equal(got, got2)


def test_attention_refuses_what_its_loads_cannot_take():
    q = torch.zeros(1, 2, 1, 64, dtype=BF, device=DEV)
    n = torch.zeros(1, dtype=torch.int32, device=DEV)
    flat = torch.zeros(1 * 1 * 16 * 64 + 8, dtype=BF, device=DEV)
    ok = flat[: 16 * 64].view(1, 1, 16, 64)
    odd = flat[1 : 1 + 16 * 64].view(1, 1, 16, 64)
    with pytest.raises(ValueError, match="16-byte aligned"):
        fc.tree_attention(q, ok, odd, n)
    with pytest.raises(ValueError, match="16 bytes"):
        fc.tree_attention(q, torch.zeros(1, 1, 16, 68, dtype=BF, device=DEV)[..., :64], ok, n)
    with pytest.raises(ValueError, match="multiples of"):
        fc.tree_attention(q[..., :20], ok[..., :20], ok[..., :20], n)
    c = torch.zeros(1, 1, 16, 24, dtype=I8, device=DEV)
    s = torch.zeros(1, 1, 16, dtype=torch.uint8, device=DEV)
    with pytest.raises(ValueError, match="multiples of"):
        fc.tree_attention(q[..., :24], c, c, n, key_scales=s, value_scales=s)


def test_empty_inputs():
    e = torch.zeros(2, 4, 0, 64, dtype=BF, device=DEV)
    k = torch.zeros(2, 2, 9, 64, dtype=BF, device=DEV)
    n = torch.zeros(2, dtype=torch.int32, device=DEV)
    assert fc.tree_attention(e, k, k, n).shape == (2, 4, 0, 64)
    out, lse = fc.tree_attention(torch.ones(2, 4, 3, 64, dtype=BF, device=DEV), k[:, :, :0], k[:, :, :0], n, return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    assert fc.kv_cache_read(k, k, n=0)[0].shape == (2, 2, 0, 64)
    fc.kv_cache_append(e[:, :2], e[:, :2], k, k.clone(), n)
    a, b = fc.qk_norm_rope(e, e, torch.zeros(0, dtype=torch.int32, device=DEV), torch.zeros(32, device=DEV))
    assert a.shape == e.shape and b.shape == e.shape


# ------------------------------------------------------------------------------------- together, streams and graphs
def _step(fmt, dtype=BF, m=6):
    """A serving step's tensors: a projection's output, a cache of two sequences, their lengths."""
    g = torch.Generator().manual_seed(11)
    b, hq, h, d, n = 2, 8, 2, 64, 700
    x = torch.randn(b, m, hq + 2 * h, d, generator=g).to(dtype).to(DEV).transpose(1, 2)
    _, cache, _ = _make(b, hq, h, m, n, d, fmt, dtype, seed=12)
    lens = torch.tensor([640, 55], device=DEV, dtype=torch.int32)
    w = (1 + 0.1 * torch.randn(2, d, generator=g)).to(dtype).to(DEV)
    return x, cache, lens, w, _freq(d).to(DEV), _tree(b, m, seed=1).to(DEV), (b, hq, h, m, d, n)


def _serve(x, cache, lens, w, freq, mask, hq, h, m):
    pos = lens[:, None] + torch.arange(m, device=DEV, dtype=torch.int32)
    q, k = fc.qk_norm_rope(x[:, :hq], x[:, hq : hq + h], pos, freq, w[0], w[1])
    fc.kv_cache_append(k, x[:, hq + h :], cache[0], cache[1], lens, cache[2], cache[3])
    out, lse = fc.tree_attention(q, cache[0], cache[1], lens, mask, key_scales=cache[2], value_scales=cache[3], return_lse=True)
    return q, out, lse


@pytest.mark.parametrize("fmt", ["16", FP8, I8])
def test_a_serving_step_and_the_pruning_of_its_cache(fmt):
    """Norm and rotation, append, attention; then the column reduction over the cached keys, its top-k, the kept positions
    in a smaller cache, and attention over that."""
    x, cache, lens, w, freq, mask, (b, hq, h, m, d, n) = _step(fmt)
    q, out, lse = _serve(x, cache, lens, w, freq, mask, hq, h, m)
    k16, v16 = fc.kv_cache_read(*cache, dtype=BF)
    _check_attention(out, lse, q.cpu(), k16.cpu().double(), v16.cpu().double(), lens.tolist(), mask.cpu())
    keep = 32
    scores = fc.flash_colreduce(q, k16.repeat_interleave(hq // h, 1)[:, :, :50], "sum")
    _, pos = fc.topk_columns(scores.view(b, h, hq // h, 50).sum(2), keep)
    ks, vs = fc.kv_cache_read(*cache, positions=pos, dtype=BF)
    assert torch.equal(ks, k16.gather(2, pos[..., None].expand(b, h, keep, d)))
    small = [None if c is None else torch.zeros_like(c[:, :, : keep + m]) for c in cache]
    zero = torch.zeros_like(lens)
    fc.kv_cache_append(ks, vs, small[0], small[1], zero, small[2], small[3])
    back = fc.kv_cache_read(*small, n=keep, dtype=BF)
    assert torch.equal(back[0], ks) and torch.equal(back[1], vs)  # what a cache held is written without a change
    kept = zero + keep
    q2, out2, lse2 = _serve(x, small, kept, w, freq, mask, hq, h, m)
    k2, v2 = fc.kv_cache_read(*small, dtype=BF)
    _check_attention(out2, lse2, q2.cpu(), k2.cpu().double(), v2.cpu().double(), kept.tolist(), mask.cpu())


@pytest.mark.parametrize("fmt", ["16", FP8, I8])
def test_captured_steps_follow_new_lengths_and_inputs(fmt):
    x, cache, lens, w, freq, mask, (b, hq, h, m, d, n) = _step(fmt)
    _serve(x, [None if c is None else c.clone() for c in cache], lens, w, freq, mask, hq, h, m)  # first calls are made outside a capture
    torch.cuda.synchronize()
    graphs, outs = [], []
    state = [[None if c is None else c.clone() for c in cache] for _ in range(2)]
    for i in range(2):  # two graphs live at once
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_serve(x, state[i], lens, w, freq, mask, hq, h, m))
        graphs.append(graph)
    for new in ([640, 55], [0, 300], [127, 694], [128, 1]):
        lens.copy_(torch.tensor(new, dtype=torch.int32))
        x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(new[0])).to(x.dtype))
        for i in range(2):
            graphs[i].replay()
        fresh = [None if c is None else c.clone() for c in cache]
        want = _serve(x, fresh, lens, w, freq, mask, hq, h, m)
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(a, e) for a, e in zip(outs[i], want))
        for j in range(4):
            if cache[j] is not None:
                for s in state:
                    cache_now = _bits(s[j])
                    at = new
                    for bb in range(b):
                        assert torch.equal(cache_now[bb, :, at[bb] : at[bb] + m], _bits(fresh[j])[bb, :, at[bb] : at[bb] + m])
                    s[j].view(torch.uint8).copy_(cache[j].view(torch.uint8))


def test_two_streams_at_once():
    x, cache, lens, w, freq, mask, (b, hq, h, m, d, n) = _step(FP8)
    want = _serve(x, cache, lens, w, freq, mask, hq, h, m)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                mine = [c.clone() for c in cache]
                got[i].append(_serve(x, mine, lens, w, freq, mask, hq, h, m))
    torch.cuda.synchronize()
    for i in range(2):
        for r in got[i]:
            assert all(torch.equal(a, e) for a, e in zip(r, want))


def test_a_long_cache_passes_32_bit_offsets():
    """More than 2^31 values in front of the last sequence's positions, in every format."""
    b, h, n, d = 5, 8, 131072 * 4, 128
    for fmt in (I8, BF):
        cache = [torch.zeros((b, h, n, d), dtype=fmt, device=DEV) for _ in range(2)]
        scales = [torch.full((b, h, n), 127, dtype=torch.uint8, device=DEV) for _ in range(2)] if fmt == I8 else [None, None]
        g = torch.Generator().manual_seed(2)
        k, v = (torch.randn(b, h, 3, d, generator=g).to(BF) for _ in range(2))
        lens = torch.tensor([0, 5, 2 ** 18, n - 100, n - 3], device=DEV)
        fc.kv_cache_append(k.to(DEV), v.to(DEV), cache[0], cache[1], lens, *scales)
        sel = (lens[:, None, None] + torch.arange(3, device=DEV)).expand(b, h, 3)
        rk, rv = fc.kv_cache_read(*cache, *scales, positions=sel, dtype=BF)
        if fmt == BF:
            assert torch.equal(rk.cpu(), k) and torch.equal(rv.cpu(), v)
        else:
            assert torch.equal(rv.cpu().double(), dequantize_rows(*quantize_rows(v, I8)))
        # attention over the last 100 positions of the last two sequences: the view starts beyond 2^31 values
        part = [None if c is None else c[3:, :, n - 256 :] for c in (*cache, *scales)]
        q = torch.randn(2, h, 3, d, generator=g).to(BF)
        got, lse = fc.tree_attention(q.to(DEV), part[0], part[1], torch.tensor([156, 253], device=DEV), key_scales=part[2],
                                     value_scales=part[3], return_lse=True)
        kk, vv = fc.kv_cache_read(*[None if c is None else c.contiguous() for c in part], dtype=BF)
        _check_attention(got, lse, q, kk.cpu().double(), vv.cpu().double(), [156, 253], None)
        # and over everything in front of them: keys of zeros, so each weight is 1 / (n - 3 + ...)
        full = fc.tree_attention(q.to(DEV), cache[0][3:], cache[1][3:], torch.tensor([n - 100, n - 3], device=DEV),
                                 key_scales=None if fmt == BF else scales[0][3:], value_scales=None if fmt == BF else scales[1][3:], return_lse=True)[1]
        assert (full > math.log(n - 100)).all() and (full < math.log(n) + 0.2).all()
        del cache, scales, part


def test_another_device_than_the_current_one():
    if torch.cuda.device_count() < 2:
        pytest.skip("needs two GPUs")
    x, cache, lens, w, freq, mask, (b, hq, h, m, d, n) = _step(I8)
    want = _serve(x, cache, lens, w, freq, mask, hq, h, m)
    with torch.cuda.device(1):
        got = _serve(x, cache, lens, w, freq, mask, hq, h, m)
    assert all(torch.equal(a, e) for a, e in zip(got, want))


@pytest.mark.parametrize("fmt", ["16", FP8])
@pytest.mark.parametrize("hq,h,m,n,d", [(24, 1, 3, 130, 128), (9, 3, 32, 100, 64), (32, 32, 70, 128, 128), (10, 5, 64, 700, 64), (64, 16, 20, 140, 128)])
def test_many_short_groups(fmt, hq, h, m, n, d):
    """More groups of one or two tiles than CTAs, 65 to 128 rows each: a warpgroup has no tile in every other group."""
    b = 40
    g = torch.Generator().manual_seed(n)
    lens = torch.randint(0, n - m + 1, (b,), generator=g).tolist()
    q, cache, x = _make(b, hq, h, m, n, d, fmt, BF, seed=n)
    got, lse = _run(q, cache, lens)
    pick = [0, 17, b - 1]
    _check_attention(got[pick], lse[pick], q[pick], x[0][pick], x[1][pick], [lens[i] for i in pick], None)
    # every sequence alone gives the same up to the order in which partial sums are added
    one, _ = _run(q[5:6], [None if c is None else c[5:6] for c in cache], lens[5:6])
    assert (one.float() - got[5:6].float()).abs().max() <= 4 * _u(BF) * x[1].abs().max()


# ----------------------------------------------------------------------------------------------- expired bounded waits
@pytest.mark.parametrize("skip", [0, 3])
@pytest.mark.parametrize("fmt", ["16", I8])
@pytest.mark.parametrize("hq,h,m,d", [(4, 1, 1, 128), (4, 1, 8, 64), (4, 1, 16, 128), (4, 1, 24, 128), (4, 1, 64, 128)])
def test_an_expired_wait_is_reported_and_the_next_call_is_right(skip, fmt, hq, h, m, d, monkeypatch):
    """Every attention kernel with one tile's load left out (nothing is in flight for its slot) and waits of a millisecond: the
    CTA gives up in an orderly way, the status reaches the host, and the call after the one that reports it runs."""
    import ctypes as C

    from flash_colreduce_b200 import _native as nat

    monkeypatch.setenv("FCR_DEBUG_SYNC", "0")
    q, cache, x = _make(1, hq, h, m, 2000, d, fmt, BF, seed=m)
    before, lse = _run(q, cache, [2000 - m])
    torch.cuda.synchronize()
    nat.check(nat.lib.fcr_self_test_hooks(2_000_000, skip), "fcr_self_test_hooks")
    try:
        _run(q, cache, [2000 - m])
    finally:
        nat.check(nat.lib.fcr_self_test_hooks(0, -1), "fcr_self_test_hooks")
    torch.cuda.synchronize()
    code = C.c_int32(-1)
    rc = nat.lib.fcr_poll_device_status(C.byref(code))
    # 16 tiles on 16 CTAs: CTA 0 has one tile of a 16-bit cache (load 0), two loads of an 8-bit one (0 and 1)
    if skip == 0:
        assert rc == nat.FCR_ERR_DEVICE_TIMEOUT and 71 <= code.value <= 92, (rc, code.value)
    else:
        assert rc == nat.FCR_OK
    after, lse2 = _run(q, cache, [2000 - m])
    assert torch.equal(before, after) and torch.equal(lse, lse2)


def test_the_next_attention_call_raises_for_the_failed_one(monkeypatch):
    from flash_colreduce_b200 import _native as nat

    monkeypatch.setenv("FCR_DEBUG_SYNC", "0")
    q, cache, x = _make(1, 4, 1, 2, 2000, 128, "16", BF)
    want, _ = _run(q, cache, [1998])
    nat.check(nat.lib.fcr_self_test_hooks(2_000_000, 0), "fcr_self_test_hooks")
    try:
        _run(q, cache, [1998])
    finally:
        nat.check(nat.lib.fcr_self_test_hooks(0, -1), "fcr_self_test_hooks")
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="status 4.*earlier call"):
        _run(q, cache, [1998])
    got, _ = _run(q, cache, [1998])
    assert torch.equal(got, want)


def test_repeated_signatures_with_unaligned_queries_and_other_types():
    """A signature that was checked once: the same shapes at an unaligned base, other types of lengths, scales as bytes."""
    q, cache, x = _make(2, 4, 2, 3, 300, 64, I8, BF, seed=21)
    lens = torch.tensor([290, 17], device=DEV)
    want = fc.tree_attention(q.to(DEV), cache[0], cache[1], lens, key_scales=cache[2], value_scales=cache[3])
    flat = torch.empty(q.numel() + 1, dtype=BF, device=DEV)
    odd = flat[1:].view(q.shape)
    odd.copy_(q)
    for _ in range(2):
        assert torch.equal(fc.tree_attention(odd, cache[0], cache[1], lens, key_scales=cache[2], value_scales=cache[3]), want)
        assert torch.equal(fc.tree_attention(q.to(DEV), cache[0], cache[1], lens.int(), key_scales=cache[2].view(torch.uint8),
                                             value_scales=cache[3].view(torch.uint8)), want)
    with pytest.raises(ValueError, match="lengths"):
        fc.tree_attention(q.to(DEV), cache[0], cache[1], lens.float(), key_scales=cache[2], value_scales=cache[3])
    leaf = q.to(DEV).requires_grad_()
    with pytest.raises(RuntimeError, match="no backward pass"):
        fc.tree_attention(leaf, cache[0], cache[1], lens, key_scales=cache[2], value_scales=cache[3])
    with torch.no_grad():
        assert torch.equal(fc.tree_attention(leaf, cache[0], cache[1], lens, key_scales=cache[2], value_scales=cache[3]), want)


def test_the_rows_are_quantised_alike_wherever_they_lie():
    """Appending a prompt at once, in pieces, or token by token leaves the same bits."""
    g = torch.Generator().manual_seed(31)
    k, v = (torch.randn(2, 3, 70, 96, generator=g).to(HF).to(DEV) for _ in range(2))
    caches = [_empty_cache(2, 3, 80, 96, FP8) for _ in range(3)]
    start = torch.tensor([0, 5], device=DEV, dtype=torch.int32)
    for c, sizes in zip(caches, ([70], [33, 1, 36], [1] * 70)):
        at = 0
        for s in sizes:
            fc.kv_cache_append(k[:, :, at : at + s], v[:, :, at : at + s], c[0], c[1], start + at, c[2], c[3])
            at += s
    for c in caches[1:]:
        assert all(torch.equal(_bits(a), _bits(b)) for a, b in zip(c, caches[0]))


@pytest.mark.parametrize("fmt", ["16", FP8, I8])
@pytest.mark.parametrize("m,g", [(1, 4), (6, 8), (12, 4), (30, 4), (64, 8)])
def test_a_nan_among_the_cached_positions_reaches_every_row(fmt, m, g):
    """Every row attends every cached position: a key or value that is NaN makes the rows of its head NaN, and no others."""
    for which in (0, 1):
        q, cache, x = _make(2, 2 * g, 2, m, 300, 64, fmt, BF, seed=3)
        if fmt == "16":
            cache[which][0, 1, 40, 5] = float("nan")
        else:
            cache[2 + which].view(torch.uint8)[0, 1, 40] = 255
        got, lse = _run(q, cache, [200, 230])
        clean = torch.ones(2, 2 * g, dtype=torch.bool)
        clean[0, g:] = False
        assert torch.isfinite(got[clean.to(DEV)].float()).all()
        bad = got[0, g:]
        assert (bad[..., 5].isnan().all() if which and fmt == "16" else bad.isnan().all())
        assert lse[0, g:].isnan().all() == (which == 0)


def test_options_given_as_tensors_are_read_anew():
    q, cache, x = _make(1, 2, 1, 2, 200, 64, "16", HF)
    scale = torch.tensor(0.1)
    a, _ = _run(q, cache, [190], scale=scale)
    scale.fill_(0.3)
    b, _ = _run(q, cache, [190], scale=scale)
    _check_attention(a, None, q, x[0], x[1], [190], None, 0.1)
    _check_attention(b, None, q, x[0], x[1], [190], None, 0.3)
