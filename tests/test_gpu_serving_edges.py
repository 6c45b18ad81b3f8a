"""The attention of drafted tokens where its kernels' warps, types and lengths meet an edge (needs a B200).

Tolerances are those of test_gpu_serving.py; what a test adds to them is derived beside it.
"""
import ctypes as C
import math

import pytest
import torch

import flash_colreduce_b200 as fc
from flash_colreduce_b200 import _native as nat
from oracle.serving_oracle import attention, dequantize_rows, quantize_rows
from test_gpu_serving import BF, DEV, FP8, HF, I8, _bits, _check_attention, _empty_cache, _make, _run, _tree
from test_serving_edges_cpu import status_codes

pytestmark = pytest.mark.gpu


def _check_strictly(got, lse, q, k, v, lens, mask, scale=None):
    """As ``_check_attention``, and infinite entries of the output and of the log-sum-exp are equal with their signs."""
    _check_attention(got, lse, q, k, v, lens, mask, scale)
    want, want_lse, _ = attention(q, k, v, lens, mask, scale)
    for g, w in ((got.cpu().double(), want), (lse.cpu().double(), want_lse)):
        assert torch.equal(g.isinf(), w.isinf()) and torch.equal(g[w.isinf()], w[w.isinf()])


# --------------------------------------------------------------------------- warps of which only some lanes hold a row
@pytest.mark.parametrize("fmt", ["16", FP8])
@pytest.mark.parametrize("have", [60, 2900])  # one CTA has all of a head's keys; several share them
@pytest.mark.parametrize("hq,h,m,d", [
    (10, 2, 7, 128), (8, 2, 5, 64), (6, 2, 13, 128), (3, 1, 27, 80), (3, 1, 41, 64), (7, 1, 26, 128), (10, 2, 67, 64),
])
def test_warps_that_hold_fewer_rows_than_lanes(fmt, have, hq, h, m, d):
    """35, 20, 39, 81, 123, 182 and 335 rows per key head: lanes without a row leave the epilogue early, the others write
    statistics and put non-finite drafted values back."""
    q, cache, x = _make(1, hq, h, m, have + m + 3, d, fmt, HF, seed=m)
    mask = _tree(1, m, seed=m)
    mask[0, : m // 2, 2:5] = False
    mask[0, m // 2 :, 2] = True
    mask[0, m - 1, 4] = True
    for head, token, col, value in ((0, 2, 3, math.nan), (0, 2, 7, -math.inf), (0, 2, 12, math.inf), (h - 1, 4, 7, math.inf)):
        if fmt == "16":
            cache[1][0, head, have + token, col] = value
            x[1][0, head, have + token, col] = value
    if fmt == FP8:
        cache[3].view(torch.uint8)[0, 0, have + 2] = 255
        x[1][0, 0, have + 2] = math.nan
    got, lse = _run(q, cache, [have], mask)
    _check_strictly(got, lse, q, x[0], x[1], [have], mask)
    again, lse2 = _run(q, cache, [have], mask)
    assert torch.equal(got.nan_to_num(7.0), again.nan_to_num(7.0)) and torch.equal(lse, lse2)


@pytest.mark.parametrize("m", [1, 5, 16])
def test_column_reduction_with_a_score_cache_and_lanes_without_a_query(m):
    """Few queries and long keys: the key-streaming rows pass keeps its scores; lanes beyond the last query keep none."""
    g = torch.Generator().manual_seed(m)
    q, k = torch.randn(2, 3, m, 128, generator=g).to(BF), torch.randn(2, 3, 5000, 128, generator=g).to(BF)
    got = fc.flash_colreduce(q.to(DEV), k.to(DEV), "sum")
    want = torch.softmax(q.double() @ k.double().transpose(-1, -2) / math.sqrt(128), -1).sum(2)
    # the operator's bar: 2e-3 relative and 1e-5, and one rounding to bf16
    assert ((got.cpu().double() - want).abs() <= 1e-5 + (2e-3 + 2.0 ** -8) * want.abs()).all()


# ------------------------------------------------------------------------------------- fp16 weights far below the largest
@pytest.mark.parametrize("fmt", ["16", FP8, I8])
@pytest.mark.parametrize("m,g", [(1, 4), (6, 4), (8, 8), (20, 4), (40, 4)])  # every form of the kernels
@pytest.mark.parametrize("gap,first", [(14.0, True), (17.0, True), (17.5, False), (20.0, True)])
def test_a_strong_key_and_many_weak_ones_in_fp16(fmt, m, g, gap, first):
    """One key `gap` nats above 16384 others and with value 0: the output is what the others' weights, 2^-20 to 2^-30 of its
    own, add up to.

    A weight is rounded to fp16 once, by half a step: u of itself, or 2^-25 below 2^-14.  The row's largest weight in a CTA
    is 2^7 at least, so that each key adds at most 2^-32 of the row's sum times its value to the usual bound.
    """
    heads, n, d = 148, 16384, 64  # a head per CTA
    at = 0 if first else n - 1
    gen = torch.Generator().manual_seed(m)
    k, v = torch.zeros(n + m, d), torch.empty(n + m, d)
    k[:, 1] = 0.5 * torch.rand(n + m, generator=gen)
    k[at, :2] = torch.tensor([gap, 0.0])
    v.copy_(0.5 + torch.rand(n + m, d, generator=gen))
    v[at] = 0
    q = torch.zeros(1, 1, m, d)
    q[..., :2] = 1
    q, x = q.to(HF), torch.stack([k, v]).to(HF)[:, None, None]
    if fmt == "16":
        one, values = [x[0], x[1], None, None], x.double()
    else:
        one, values = [None] * 4, []
        for i in range(2):
            codes, bits = quantize_rows(x[i], fmt)
            one[i], one[2 + i] = codes.to(fmt), bits
            values.append(dequantize_rows(codes, bits))
    cache = []
    for c in one:
        if c is None:
            cache.append(None)
            continue
        raw = c.view({2: torch.int16, 1: torch.uint8}[c.element_size()]).to(DEV)
        cache.append(raw.expand(1, heads, *raw.shape[2:]).contiguous().view(c.dtype))
    got, lse = _run(q.expand(1, heads * g, m, d), cache, [n], scale=1.0)
    want, want_lse, weight = attention(q, values[0], values[1], [n], None, 1.0)
    u = 2.0 ** -11
    big = gap + 1.0
    score = big * (d / 16 + 4) * 2.0 ** -22 + big * 2.0 ** -23 + 2.0 ** -21
    bound = u * want.abs() + 2 * (u + score) * weight + n * 2.0 ** -32 * values[1].abs().max() + 2.0 ** -24
    worst = ((got.cpu().double() - want).abs() / bound).max().item()
    assert worst <= 1.0, worst
    assert ((lse.cpu().double() - want_lse).abs() <= score + 2.0 ** -22 * want_lse.abs() + 2.0 ** -20).all()


@pytest.mark.parametrize("fmt,hq,m", [("16", 4, 1), (I8, 4, 16), ("16", 4, 24), (I8, 4, 64)])
def test_an_expired_wait_has_a_code_of_the_attention_kernels(fmt, hq, m, monkeypatch):
    """One tile's load is left out and waits last a millisecond: the code that reaches the host is of no other kernel."""
    own = {code for name, code in status_codes() if name.startswith(("ST_TR_", "ST_TD_"))}
    own -= {code for name, code in status_codes() if not name.startswith(("ST_TR_", "ST_TD_"))}
    monkeypatch.setenv("FCR_DEBUG_SYNC", "0")
    q, cache, x = _make(1, hq, 1, m, 2000, 128, fmt, BF, seed=m)
    before, lse = _run(q, cache, [2000 - m])
    torch.cuda.synchronize()
    nat.check(nat.lib.fcr_self_test_hooks(2_000_000, 0), "fcr_self_test_hooks")
    try:
        _run(q, cache, [2000 - m])
    finally:
        nat.check(nat.lib.fcr_self_test_hooks(0, -1), "fcr_self_test_hooks")
    torch.cuda.synchronize()
    code = C.c_int32(-1)
    assert nat.lib.fcr_poll_device_status(C.byref(code)) == nat.FCR_ERR_DEVICE_TIMEOUT
    assert code.value in own, code.value
    after, lse2 = _run(q, cache, [2000 - m])
    assert torch.equal(before, after) and torch.equal(lse, lse2)


@pytest.mark.parametrize("fmt", ["16", FP8, I8])
@pytest.mark.parametrize("m,g,d", [(1, 4, 128), (6, 4, 64), (8, 8, 128), (20, 4, 64), (150, 4, 128)])
@pytest.mark.parametrize("masked", [False, True])
def test_a_sequence_of_negative_length_has_no_positions(fmt, m, g, d, masked):
    """The append leaves its tokens out, and the attention attends nothing: not what lies at the first positions either."""
    n = 700
    q, cache, x = _make(4, g, 1, m, n, d, fmt, BF, seed=m)
    for i in range(2):
        if fmt == "16":
            cache[i][1, :, :] = math.nan
        else:
            cache[2 + i].view(torch.uint8)[1] = 255
    before = [None if c is None else _bits(c).clone() for c in cache]
    lens = [500, -1, 3, -(2 ** 31)]
    new = torch.ones(4, 1, m, d, dtype=BF, device=DEV)
    fc.kv_cache_append(new, new, cache[0], cache[1], torch.tensor(lens, device=DEV), cache[2], cache[3])
    for c, old in zip(cache, before):
        assert c is None or (torch.equal(_bits(c)[1::2], old[1::2]) and not torch.equal(_bits(c)[::2], old[::2]))
    mask = _tree(4, m, seed=2) if masked else None
    got, lse = _run(q, cache, lens, mask)
    assert (got[1::2] == 0).all() and (lse[1::2] == -math.inf).all()
    k, v = fc.kv_cache_read(*cache, dtype=BF)
    pick = [0, 2]
    _check_strictly(got[pick], lse[pick], q[pick], k.cpu().double()[pick], v.cpu().double()[pick], [lens[i] for i in pick],
                    None if mask is None else mask[pick])
    want, want_lse, _ = attention(q, k.cpu().double(), v.cpu().double(), lens, mask)
    assert (want[1::2] == 0).all() and (want_lse[1::2] == -math.inf).all()


# --------------------------------------------------------------------------------------------------------- autograd
@pytest.mark.parametrize("fmt", [BF, FP8])
def test_an_append_raises_the_versions_of_what_it_writes(fmt):
    """A cache that an earlier operation saved for its backward pass cannot change unnoticed."""
    cache = _empty_cache(2, 2, 20, 64, fmt)
    new = torch.randn(2, 2, 3, 64, device=DEV).to(BF)
    lens = torch.tensor([4, 5], device=DEV)
    given = [new, lens, *[c for c in cache if c is not None]]
    before = [x._version for x in given]
    fc.kv_cache_append(new, new, cache[0], cache[1], lens, cache[2], cache[3])
    assert [x._version > v for x, v in zip(given, before)] == [False, False] + [True] * (len(given) - 2)
    before = [x._version for x in given]
    fc.kv_cache_append(new[:, :, :0], new[:, :, :0], cache[0], cache[1], lens, cache[2], cache[3])  # nothing to write
    fc.kv_cache_read(*cache, dtype=BF)
    assert [x._version for x in given] == before
    if fmt == BF:
        weight = torch.ones(2, 2, 20, 64, dtype=BF, device=DEV, requires_grad=True)
        cache[1].zero_()
        for part in (cache[1], cache[1][:, :, 8:]):  # saved whole, and as a view
            loss = (weight[:, :, -part.shape[2] :] * part).sum()
            fc.kv_cache_append(new, new, cache[0], cache[1], lens)
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                loss.backward()
    with torch.inference_mode():  # whose tensors have no versions
        mine = [None if c is None else c.clone() for c in cache]
        fc.kv_cache_append(new, new, mine[0], mine[1], lens, mine[2], mine[3])
        got = fc.kv_cache_read(*mine, dtype=BF)
    assert torch.equal(got[0][0, :, 4:7], fc.kv_cache_read(*cache, dtype=BF)[0][0, :, 4:7])


# ------------------------------------------------------------------------------------- codes and scales at every size
@pytest.mark.parametrize("fmt", [FP8, I8])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("d", [64, 33])
def test_rows_of_every_scale_are_read_in_either_type(fmt, dtype, d):
    """All 256 scale bytes by all 256 codes, read in the type they were not written from too: one rounding of code * 2^e."""
    codes = torch.arange(256).repeat(256, 1).to(torch.uint8)
    codes = torch.cat([codes, codes[:, : -256 % d]], 1).view(256, -1, d).transpose(0, 1)[None].contiguous()  # (1, heads, 256 scales, d)
    scales = torch.arange(256).to(torch.uint8).expand(codes.shape[:3]).contiguous()
    data = codes.to(DEV).view(fmt)
    got = fc.kv_cache_read(data, data, scales.to(DEV), scales.to(DEV), dtype=dtype)
    want = dequantize_rows(codes.view(fmt), scales).to(dtype)
    for g in got:
        assert torch.equal(g.cpu().isnan(), want.isnan()) and torch.equal(g.cpu().nan_to_num(3.0, 7.0, -7.0), want.nan_to_num(3.0, 7.0, -7.0))


def _scaled(b, hq, h, m, n, d, fmt, dtype, shifts, seed):
    """Queries and a cache of 8 bits whose rows' exponents are moved by one of `shifts` (keys, values); the values as read."""
    q, cache, _ = _make(b, hq, h, m, n, d, fmt, dtype, seed=seed)
    g = torch.Generator().manual_seed(seed)
    for i in range(2):
        by = torch.tensor(shifts[i])[torch.randint(0, len(shifts[i]), (b, h, n), generator=g)]
        by[:, :, 128:256] = 0  # a tile of ordinary scales
        bits = cache[2 + i].view(torch.uint8)
        bits.copy_((bits.cpu().int() + by).to(torch.uint8))
    return q, cache


@pytest.mark.parametrize("fmt", [FP8, I8])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("m,g,d", [(1, 4, 128), (6, 4, 80), (8, 8, 64), (20, 4, 128), (40, 4, 64)])
def test_attention_over_finite_scales_of_any_size(fmt, dtype, m, g, d):
    """Scales far outside 2^-24 .. 2^5, beside ordinary ones in the same tile and alone."""
    for shifts in (((0, -40, -100), (0, 8, -26)) if dtype is HF else ((0, -40, -100), (0, 60, -60)), ((-30,), (-20,)), ((0,), (7,))):
        q, cache = _scaled(2, 2 * g, 2, m, 600, d, fmt, dtype, shifts, seed=m)
        lens = [600 - m, 300]
        mask = _tree(2, m, seed=3)
        got, lse = _run(q, cache, lens, mask)
        k, v = (x.cpu().double() for x in fc.kv_cache_read(*cache, dtype=dtype))
        assert torch.isfinite(v).all()
        _check_strictly(got, lse, q, k, v, lens, mask)


@pytest.mark.parametrize("fmt", [FP8, I8])
@pytest.mark.parametrize("m,g,d", [(1, 4, 128), (6, 4, 80), (8, 8, 64), (20, 4, 128), (40, 4, 64)])
def test_values_that_fp16_cannot_hold_are_infinite(fmt, m, g, d):
    """Attention in fp16 over rows written from bf16: such a value is read as an infinity, by the rows that attend it."""
    q, cache, _ = _make(2, 2 * g, 2, m, 600, d, fmt, HF, seed=m)
    lens = [600 - m, 300]
    one = torch.full((1, 1, 1, d), 1.0, dtype=BF, device=DEV)
    one[..., 1::2] = -1
    zero = torch.zeros_like(one)
    for row, at, value in ((0, 40, one * 1e6 * (torch.arange(d, device=DEV) == 5)), (1, 300 + m // 2, one * 3e5)):
        part = [c[row : row + 1, 1:] for c in cache]
        fc.kv_cache_append(zero, value.to(BF), part[0], part[1], torch.tensor([at], device=DEV), part[2], part[3])
    mask = _tree(2, m, seed=3)
    got, lse = _run(q, cache, lens, mask)
    k, v = (x.cpu().double() for x in fc.kv_cache_read(*cache, dtype=HF))
    assert v[0, 1, 40, 5] == -math.inf and v[0, 1, 40].isinf().sum() == 1 and v[1, 1, 300 + m // 2].isinf().all()
    _check_strictly(got, lse, q, k, v, lens, mask)
    assert (got[0, g:, :, 5] == -math.inf).all()


@pytest.mark.parametrize("fmt", ["16", FP8, I8])
@pytest.mark.parametrize("m,g", [(1, 4), (6, 8), (12, 4), (30, 4), (64, 8)])
def test_a_nan_among_the_cached_positions_leaves_the_rest_as_it_is(fmt, m, g):
    """What it must not reach is compared with the oracle: other heads, other columns, and the log-sum-exp for a value."""
    lens = [200, 230]
    for which in (0, 1):
        q, cache, x = _make(2, 2 * g, 2, m, 300, 64, fmt, BF, seed=3)
        if fmt == "16":
            cache[which][0, 1, 40, 5] = math.nan
            x[which][0, 1, 40, 5] = math.nan
        else:
            cache[2 + which].view(torch.uint8)[0, 1, 40] = 255
            x[which][0, 1, 40] = math.nan
        got, lse = _run(q, cache, lens)
        _check_strictly(got, lse, q, x[0], x[1], lens, None)
        hit = torch.zeros(2, 2 * g, dtype=torch.bool, device=DEV)
        hit[0, g:] = True
        assert torch.isfinite(lse[~hit]).all() and torch.isfinite(got[~hit].float()).all()
        assert torch.isfinite(lse[hit]).all() if which else lse[hit].isnan().all()
        assert got[hit][..., 5].isnan().all() and got[hit][..., 6].isnan().all() == (fmt != "16" or which == 0)
