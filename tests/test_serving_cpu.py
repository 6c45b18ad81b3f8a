"""The serving operators without a GPU: refusals of the Python and the C entry points, and the oracle against itself."""
import ctypes as C

import pytest
import torch

import flash_colreduce_b200 as fc
from flash_colreduce_b200 import _native as nat
from oracle.serving_oracle import attention, dequantize_rows, quantize_rows, rope

H16 = torch.float16


def _cache(b=2, h=2, n=16, d=32, fmt=torch.int8):
    c = torch.zeros(b, h, n, d).to(fmt)
    s = torch.zeros(b, h, n, dtype=torch.uint8)
    return c, c.clone(), s, s.clone()


def test_cpu_tensors_are_refused():
    x = torch.zeros(1, 2, 3, 16, dtype=H16)
    n = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="must be on a CUDA device"):
        fc.qk_norm_rope(x, x, torch.arange(3), torch.zeros(8))
    with pytest.raises(ValueError, match="must be on a CUDA device"):
        fc.kv_cache_append(x, x, x.clone(), x.clone(), n)
    with pytest.raises(ValueError, match="must be on a CUDA device"):
        fc.kv_cache_read(x, x)
    with pytest.raises(ValueError, match="must be on a CUDA device"):
        fc.tree_attention(x, x, x, n)


@pytest.mark.parametrize("change,error,text", [
    (dict(key=torch.zeros(2, 1, 3, 17, dtype=H16)), ValueError, "same B, M and D"),
    (dict(key=torch.zeros(2, 1, 3, 16)), TypeError, "one dtype"),
    (dict(query=torch.zeros(2, 4, 3, 16, dtype=torch.float64), key=torch.zeros(2, 1, 3, 16, dtype=torch.float64)), TypeError, "fp16, bf16 or fp32"),
    (dict(query=torch.zeros(2, 4, 3, 264, dtype=H16), key=torch.zeros(2, 1, 3, 264, dtype=H16)), ValueError, "exceeds 256"),
    (dict(inv_freq=torch.zeros(9)), ValueError, "inv_freq"),
    (dict(inv_freq=torch.zeros(8, dtype=H16)), ValueError, "inv_freq"),
    (dict(positions=torch.arange(4)), ValueError, "positions"),
    (dict(positions=torch.zeros(3)), ValueError, "positions"),
    (dict(q_weight=torch.zeros(15, dtype=H16)), ValueError, "weights"),
    (dict(q_weight=torch.zeros(16, dtype=torch.bfloat16)), ValueError, "weights"),
    (dict(q_weight=torch.zeros(16), k_weight=torch.zeros(16, dtype=H16)), ValueError, "weights"),
    (dict(q_weight=torch.zeros(16, dtype=H16, requires_grad=True)), RuntimeError, "no backward pass"),
])
def test_rope_refusals(change, error, text):
    args = dict(query=torch.zeros(2, 4, 3, 16, dtype=H16), key=torch.zeros(2, 1, 3, 16, dtype=H16), positions=torch.arange(3),
                inv_freq=torch.zeros(8))
    with pytest.raises(error, match=text):
        fc.qk_norm_rope(**{**args, **change})


@pytest.mark.parametrize("change,error,text", [
    (dict(value=torch.zeros(2, 2, 3, 32, dtype=torch.bfloat16)), TypeError, "one dtype"),
    (dict(key=torch.zeros(2, 2, 3, 32), value=torch.zeros(2, 2, 3, 32)), TypeError, "fp16 or bf16"),
    (dict(key=torch.zeros(2, 1, 3, 32, dtype=H16), value=torch.zeros(2, 1, 3, 32, dtype=H16)), ValueError, "must be"),
    (dict(value=torch.zeros(2, 2, 4, 32, dtype=H16)), ValueError, "must be"),
    (dict(lengths=torch.zeros(2)), ValueError, "lengths"),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), ValueError, "lengths"),
    (dict(counts=torch.zeros(2, dtype=torch.int64)), ValueError, "counts"),
    (dict(key_scales=None), ValueError, "key_scales"),
    (dict(value_scales=torch.zeros(2, 2, 15, dtype=torch.uint8)), ValueError, "value_scales"),
    (dict(value_scales=torch.zeros(2, 2, 16)), ValueError, "value_scales"),
    (dict(key_cache=torch.zeros(2, 2, 16, 32)), TypeError, "value_cache"),
    (dict(value_cache=torch.zeros(2, 2, 17, 32, dtype=torch.int8)), ValueError, "one shape"),
    (dict(value_cache=torch.zeros(2, 2, 32, 16, dtype=torch.int8).transpose(2, 3)), ValueError, "innermost"),
    (dict(key_cache=torch.zeros(2, 1, 16, 32, dtype=torch.int8).expand(2, 2, 16, 32)), ValueError, "expanded"),
    (dict(key=torch.zeros(2, 2, 3, 32, dtype=H16, requires_grad=True)), RuntimeError, "no backward pass"),
])
def test_append_refusals(change, error, text):
    kc, vc, ks, vs = _cache()
    args = dict(key=torch.zeros(2, 2, 3, 32, dtype=H16), value=torch.zeros(2, 2, 3, 32, dtype=H16), key_cache=kc, value_cache=vc,
                lengths=torch.zeros(2, dtype=torch.int32), key_scales=ks, value_scales=vs)
    with pytest.raises(error, match=text):
        fc.kv_cache_append(**{**args, **change})


def test_a_16_bit_cache_has_one_type_and_no_scales():
    x = torch.zeros(1, 1, 4, 16, dtype=H16)
    n, s = torch.zeros(1, dtype=torch.int32), torch.zeros(1, 1, 4, dtype=torch.uint8)
    with pytest.raises(TypeError, match="its own type"):
        fc.kv_cache_append(x.bfloat16(), x.bfloat16(), x, x.clone(), n)
    with pytest.raises(TypeError, match="its own type"):
        fc.kv_cache_read(x, x, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="no scales"):
        fc.kv_cache_read(x, x, s, s)


@pytest.mark.parametrize("change,error,text", [
    (dict(positions=torch.zeros(2, 2, 3)), ValueError, "positions"),
    (dict(positions=torch.zeros(2, 1, 3, dtype=torch.int64)), ValueError, "positions"),
    (dict(positions=torch.zeros(2, 2, 3, dtype=torch.int64), n=4), ValueError, "disagree"),
    (dict(n=17), ValueError, "must lie in"),
    (dict(n=-1), ValueError, "must lie in"),
    (dict(dtype=torch.float32), TypeError, "fp16 or bf16"),
])
def test_read_refusals(change, error, text):
    kc, vc, ks, vs = _cache()
    with pytest.raises(error, match=text):
        fc.kv_cache_read(kc, vc, ks, vs, **change)


@pytest.mark.parametrize("change,error,text", [
    (dict(query=torch.zeros(2, 3, 5, 32, dtype=H16)), ValueError, "multiple of 2"),
    (dict(query=torch.zeros(1, 4, 5, 32, dtype=H16)), ValueError, "query must be"),
    (dict(query=torch.zeros(2, 4, 257, 32, dtype=H16)), ValueError, "exceed 256"),
    (dict(query=torch.zeros(2, 4, 5, 32)), TypeError, "fp16 or bf16"),
    (dict(tree_mask=torch.ones(5, 5)), ValueError, "tree_mask"),
    (dict(tree_mask=torch.ones(5, 4, dtype=torch.bool)), ValueError, "tree_mask"),
    (dict(tree_mask=torch.ones(3, 5, 5, dtype=torch.bool)), ValueError, "tree_mask"),
    (dict(lengths=torch.zeros(1, dtype=torch.int32)), ValueError, "lengths"),
    (dict(query=torch.zeros(2, 4, 5, 32, dtype=H16, requires_grad=True)), RuntimeError, "no backward pass"),
])
def test_attention_refusals(change, error, text):
    kc, vc, ks, vs = _cache()
    args = dict(query=torch.zeros(2, 4, 5, 32, dtype=H16), key_cache=kc, value_cache=vc, lengths=torch.zeros(2, dtype=torch.int32),
                key_scales=ks, value_scales=vs)
    with pytest.raises(error, match=text):
        fc.tree_attention(**{**args, **change})


def _c_cache(**kw):
    a = dict(B=1, H=2, N=64, D=32, format=nat.FCR_KV_INT8, dtype=nat.FCR_F16, k=(4096, 2048, 32, 1), v=(4096, 2048, 32, 1))
    a.update(kw)
    return nat.KvCache(a["B"], a["H"], a["N"], a["D"], a["format"], a["dtype"], a["k"], a["v"], (128, 64, 1), (128, 64, 1))


@pytest.mark.parametrize("cache,tree,status,text", [
    (dict(), dict(Hq=3), nat.FCR_ERR_BAD_ARG, "multiple"),
    (dict(), dict(M=257), nat.FCR_ERR_UNSUPPORTED, "exceed 256"),
    (dict(), dict(M=0), nat.FCR_ERR_BAD_ARG, "positive"),
    (dict(N=0), dict(), nat.FCR_ERR_BAD_ARG, "positive"),
    (dict(D=24), dict(), nat.FCR_ERR_UNSUPPORTED, "multiples of"),
    (dict(D=144), dict(), nat.FCR_ERR_UNSUPPORTED, "up to 128"),
    (dict(format=nat.FCR_KV_16BIT, D=20), dict(), nat.FCR_ERR_UNSUPPORTED, "multiples of"),
    (dict(k=(4096, 2048, 40, 1)), dict(), nat.FCR_ERR_UNSUPPORTED, "16 bytes"),
    (dict(v=(4096, 2048, 0, 1)), dict(), nat.FCR_ERR_UNSUPPORTED, "16 bytes"),
    (dict(v=(4096, 2048, 32, 2)), dict(), nat.FCR_ERR_UNSUPPORTED, "innermost"),
    (dict(), dict(bits=16), nat.FCR_ERR_BAD_ARG, "index_bits"),
])
def test_c_entry_refusals(cache, tree, status, text):
    c = _c_cache(**cache)
    t = nat.Tree(tree.get("Hq", 4), tree.get("M", 5), (640, 160, 32, 1), tree.get("bits", 32), (0, 5), 0.1)
    assert nat.lib.fcr_tree_workspace_bytes(C.byref(c), C.byref(t), 148) == 0
    assert text in nat.last_error()
    p = C.c_void_p(4096)  # never dereferenced: every refusal comes before any device work
    rc = nat.lib.fcr_tree_attention(C.byref(c), C.byref(t), p, p, p, p, p, p, None, p, None, p, 1 << 30, None)
    assert rc in (status, nat.FCR_ERR_BAD_ARG) and rc != nat.FCR_OK


def test_c_entries_refuse_null_and_bad_sizes():
    c = _c_cache()
    t = nat.Tree(4, 5, (640, 160, 32, 1), 32, (0, 5), 0.1)
    p, st = C.c_void_p(4096), nat.strides4((1, 1, 1, 1))
    assert nat.lib.fcr_tree_workspace_bytes(None, C.byref(t), 148) == 0
    assert nat.lib.fcr_tree_workspace_bytes(C.byref(c), C.byref(t), 148) > 0
    assert nat.lib.fcr_tree_attention(None, None, *[None] * 10, 0, None) == nat.FCR_ERR_BAD_ARG
    assert nat.lib.fcr_tree_attention(C.byref(c), C.byref(t), p, p, p, None, None, p, None, p, None, p, 1 << 30, None) == nat.FCR_ERR_BAD_ARG
    assert nat.lib.fcr_kv_append(None, p, p, p, p, p, st, p, st, 1, p, None, 32, None) == nat.FCR_ERR_BAD_ARG
    assert nat.lib.fcr_kv_append(C.byref(c), p, p, p, p, p, st, p, st, 0, p, None, 32, None) == nat.FCR_ERR_BAD_ARG
    assert nat.lib.fcr_kv_append(C.byref(c), p, p, p, p, p, st, p, st, 1, p, None, 8, None) == nat.FCR_ERR_BAD_ARG
    assert nat.lib.fcr_kv_append(C.byref(_c_cache(D=257)), p, p, p, p, p, st, p, st, 1, p, None, 32, None) == nat.FCR_ERR_UNSUPPORTED
    assert nat.lib.fcr_kv_read(C.byref(c), p, p, p, p, None, 64, 0, p, p, None) == nat.FCR_ERR_BAD_ARG
    assert nat.lib.fcr_kv_read(C.byref(_c_cache(dtype=nat.FCR_F32)), p, p, p, p, None, 64, 1, p, p, None) == nat.FCR_ERR_UNSUPPORTED
    assert nat.lib.fcr_kv_read(C.byref(_c_cache(format=9)), p, p, p, p, None, 64, 1, p, p, None) == nat.FCR_ERR_BAD_ARG
    r = nat.Rope(1, 2, 1, 3, 16, 16, (96, 48, 16, 1), (48, 48, 16, 1), nat.FCR_F16, nat.FCR_F16, 0, 32, (0, 1), 1e-6)
    assert nat.lib.fcr_qk_norm_rope(None, *[p] * 8, None) == nat.FCR_ERR_BAD_ARG
    assert nat.lib.fcr_qk_norm_rope(C.byref(r), None, *[p] * 7, None) == nat.FCR_ERR_BAD_ARG
    for field, bad in (("rotary", 15), ("rotary", 18), ("position_bits", 8), ("dtype", 7), ("weight_dtype", nat.FCR_BF16), ("D", 0)):
        r2 = nat.Rope.from_buffer_copy(r)
        setattr(r2, field, bad)
        assert nat.lib.fcr_qk_norm_rope(C.byref(r2), *[p] * 8, None) == nat.FCR_ERR_BAD_ARG, field


# ------------------------------------------------------------------------------------------------------ the oracle
@pytest.mark.parametrize("fmt", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_quantised_rows_are_exact_and_nearest(fmt, dtype):
    g = torch.Generator().manual_seed(3)
    x = (torch.randn(4000, 24, generator=g) * torch.exp(2.5 * torch.randn(4000, 1, generator=g)))
    x = x.clamp(-60000, 60000).to(dtype)
    codes, bits = quantize_rows(x, fmt)
    assert torch.equal(codes.to(fmt).double(), codes)  # codes of the format
    back = dequantize_rows(codes, bits)
    assert torch.equal(back.to(dtype).double(), back)  # reading is exact in the written type
    top = x.double().abs().amax(-1)
    err = (back - x.double()).abs()
    if fmt == torch.int8:  # half a step; the step is at most the row's largest over 63.5
        assert (err <= 0.5 * torch.ldexp(torch.ones_like(top), bits.int() - 127)[:, None]).all()
        assert (torch.ldexp(torch.ones_like(top), bits.int() - 127) <= top / 63.5).all()
    else:
        assert (err <= x.double().abs() * 2.0 ** -4 + torch.ldexp(torch.ones_like(top), bits.int() - 127)[:, None] * 2.0 ** -10).all()
    again, bits2 = quantize_rows(back.to(dtype), fmt)
    assert torch.equal(dequantize_rows(again, bits2), back)  # writing what was read changes nothing


def test_quantised_rows_at_the_ends_of_the_range():
    for dtype, fmt in [(t, f) for t in (torch.float16, torch.bfloat16) for f in (torch.float8_e4m3fn, torch.int8)]:
        big = torch.finfo(dtype).max
        tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
        x = torch.tensor([[0.0, 0.0], [big, -big], [tiny, -tiny], [1.0, float("nan")], [float("inf"), 1.0]]).to(dtype)
        codes, bits = quantize_rows(x, fmt)
        back = dequantize_rows(codes, bits)
        assert (back[0] == 0).all() and torch.isfinite(back[1].to(dtype)).all() and (back[1].abs() >= 0.9 * big).all()
        assert back[3:].isnan().all()


def test_rope_keeps_norms_and_positions_are_relative():
    g = torch.Generator().manual_seed(0)
    x, y = torch.randn(1, 1, 1, 32, generator=g), torch.randn(1, 1, 1, 32, generator=g)
    f = 10000.0 ** (-torch.arange(0, 32, 2) / 32)
    for inter in (False, True):
        a = [float((rope(x, torch.tensor([p]), f, interleaved=inter) * rope(y, torch.tensor([p + 5]), f, interleaved=inter)).sum())
             for p in (0, 17, 1000003)]
        assert max(a) - min(a) < 1e-9
        assert torch.allclose(rope(x, torch.tensor([9]), f, interleaved=inter).norm(), x.double().norm())


def test_attention_oracle_on_closed_forms():
    q = torch.zeros(1, 2, 3, 8)
    k = torch.randn(1, 1, 10, 8, generator=torch.Generator().manual_seed(1))
    out, lse, _ = attention(q, k, k, torch.tensor([4]))  # scores 0: means
    for m in range(3):
        assert torch.allclose(out[0, :, m], k[0, 0, : 5 + m].double().mean(0).expand(2, 8))
        assert torch.allclose(lse[0, :, m].exp(), torch.tensor(5.0 + m).double())
    out, lse, _ = attention(q, k, k, torch.tensor([0]), mask=torch.zeros(3, 3, dtype=torch.bool))
    assert (out == 0).all() and (lse == -float("inf")).all()


# ---------------------------------------------------------------------------------------- the attention's work items
@pytest.mark.parametrize("sms", [1, 7, 148])
@pytest.mark.parametrize("b,h,hq,m,n,lens", [
    (1, 1, 1, 1, 1, [0]), (3, 1, 8, 1, 400, [0, 1, 399]), (2, 2, 8, 64, 5000, [4000, 17]), (1, 2, 4, 200, 3000, [2900]), (5, 3, 3, 7, 1000, [990, -4, 2000, 0, 128]),
    (40, 8, 32, 1, 900, [(37 * i) % 900 for i in range(40)]), (1, 8, 32, 1, 131072, [131071]),
])
def test_every_tile_belongs_to_one_cta_and_partial_results_have_no_gaps(sms, b, h, hq, m, n, lens):
    cache = nat.KvCache(b, h, n, 128, nat.FCR_KV_16BIT, nat.FCR_BF16, (h * n * 128, n * 128, 128, 1), (h * n * 128, n * 128, 128, 1), (0, 0, 0), (0, 0, 0))
    tree = nat.Tree(hq, m, (hq * m * 128, m * 128, 128, 1), 32, (0, 0), 0.1)
    rows = hq // h * m
    row_tiles = 1 if rows <= 128 else -(-rows // 256)
    buf, host = (C.c_int32 * 10)(), (C.c_int64 * b)(*lens)
    seen, loads, parts = {}, {}, {}
    for cta in range(min(sms, b * h * row_tiles * -(-n // 128))):
        i = 0
        while nat.lib.fcr_tree_segment(C.byref(cache), C.byref(tree), sms, host, cta, i, buf) == nat.FCR_OK:
            seq, head, rt, lo, hi, tiles, slot, first, last, ctas = buf
            have = min(max(lens[seq], 0), n)
            assert tiles == -(-min(have + m, n) // 128) and 0 <= lo < hi <= tiles and rt < row_tiles
            assert (slot == -1) == (lo == 0 and hi == tiles) == (first == last)
            if slot >= 0:
                assert slot == (1 if lo == 0 else 0) and (cta, slot) not in parts
                parts[cta, slot] = (seq, head, rt)
                # what the joining kernel reads: slot 1 of the group's first CTA, slot 0 of the others
                assert first <= cta <= last and (slot == 1) == (cta == first)
            for t in range(lo, hi):
                assert (seq, head, rt, t) not in seen
                seen[seq, head, rt, t] = cta
            loads[cta] = loads.get(cta, 0) + hi - lo
            i += 1
            assert ctas <= sms
    want = sum(-(-min(min(max(x, 0), n) + m, n) // 128) for x in lens) * h * row_tiles
    assert len(seen) == want and max(loads.values()) - min(loads.values()) <= 1
    groups = {}
    for (seq, head, rt, t), cta in seen.items():
        groups.setdefault((seq, head, rt), set()).add(cta)
    for key, owners in groups.items():
        assert owners == set(range(min(owners), max(owners) + 1))


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), -float("inf"), 1e300])
def test_attention_refuses_a_scale_that_is_not_a_finite_fp32_number(scale):
    kc, vc, ks, vs = _cache()
    with pytest.raises(ValueError, match="scale"):
        fc.tree_attention(torch.zeros(2, 4, 5, 32, dtype=H16), kc, vc, torch.zeros(2, dtype=torch.int32), key_scales=ks, value_scales=vs,
                          scale=scale)
    p = nat.KvCache(2, 2, 16, 32, nat.FCR_KV_INT8, nat.FCR_F16, (1024, 512, 32, 1), (1024, 512, 32, 1), (32, 16, 1), (32, 16, 1))
    t = nat.Tree(4, 5, (640, 160, 32, 1), 32, (0, 0), scale)
    assert nat.lib.fcr_tree_workspace_bytes(C.byref(p), C.byref(t), 148) == 0
    assert "scale" in nat.last_error()


def test_attention_refuses_a_head_dimension_of_zero():
    x = torch.zeros(1, 2, 3, 0, dtype=H16)
    with pytest.raises(ValueError, match="head dimension"):
        fc.tree_attention(x, x, x.clone(), torch.zeros(1, dtype=torch.int32))
