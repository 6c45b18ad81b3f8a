"""The serving operators without a GPU: what the host decides at their edges."""
import ctypes as C
import os
import re

import pytest
import torch
from torch.autograd import forward_ad

import flash_colreduce_b200 as fc
from flash_colreduce_b200 import _native as nat
from oracle.serving_oracle import attention

CSRC = os.path.join(os.path.dirname(fc.__file__), "csrc")


def status_codes():
    """Every kernel's status codes as the sources define them: [(name, code)]."""
    found = []
    for name in sorted(os.listdir(CSRC)):
        with open(os.path.join(CSRC, name)) as f:
            found += [(n, int(c)) for n, c in re.findall(r"\b(ST_[A-Z0-9_]+)\s*=\s*(\d+)", f.read())]
    return found


def test_a_status_code_names_one_wait():
    """All kernels of a device report into one mailbox: a code must say which kernel and which wait it was."""
    found = status_codes()
    assert len(found) > 50 and len({n for n, _ in found}) == len(found)
    codes = {}
    for name, code in found:
        codes.setdefault(code, []).append(name)
    assert {c: n for c, n in codes.items() if len(n) > 1} == {}


@pytest.mark.parametrize("m", [1, 200])
def test_a_sequence_of_negative_length_takes_one_tile(m):
    """It has no positions, but somebody has to write its zeros: one tile per group, whatever the drafted tokens are."""
    b, h, n, lens = 3, 2, 1000, [-1, 300, -(2 ** 40)]
    strides = (h * n * 128, n * 128, 128, 1)
    cache = nat.KvCache(b, h, n, 128, nat.FCR_KV_16BIT, nat.FCR_BF16, strides, strides, (0, 0, 0), (0, 0, 0))
    tree = nat.Tree(h, m, (h * m * 128, m * 128, 128, 1), 32, (0, 0), 0.1)
    buf, tiles, i = (C.c_int32 * 10)(), {}, 0
    while nat.lib.fcr_tree_segment(C.byref(cache), C.byref(tree), 1, (C.c_int64 * b)(*lens), 0, i, buf) == nat.FCR_OK:
        tiles[buf[0], buf[1]] = buf[5]
        i += 1
    assert tiles == {(s, k): -(-(300 + m) // 128) if s == 1 else 1 for s in range(b) for k in range(h)}


def test_the_oracle_knows_negative_lengths():
    q = torch.zeros(2, 2, 3, 8)
    k = torch.randn(2, 1, 10, 8, generator=torch.Generator().manual_seed(1))
    out, lse, _ = attention(q, k, k, torch.tensor([-1, 0]))
    assert (out[0] == 0).all() and (lse[0] == -float("inf")).all()
    assert torch.allclose(out[1, :, 2], k[1, 0, :3].double().mean(0).expand(2, 8))


def _dual(x):
    return forward_ad.make_dual(x, torch.ones_like(x))


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("call,name", [(fc.qk_norm_rope, n) for n in ("query", "key", "inv_freq", "q_weight", "k_weight")] +
                         [(fc.kv_cache_append, n) for n in ("key", "value", "key_cache", "value_cache")] +
                         [(fc.kv_cache_read, n) for n in ("key_cache", "value_cache")] +
                         [(fc.tree_attention, n) for n in ("query", "key_cache", "value_cache")])
def test_tangents_are_refused(call, name, grad):
    """Forward-mode derivatives pass through no_grad; an input that carries one is refused like one that requires a gradient."""
    x = torch.zeros(1, 2, 3, 16, dtype=torch.float16)
    args = {fc.qk_norm_rope: dict(query=x, key=x, positions=torch.arange(3), inv_freq=torch.zeros(8), q_weight=x[0, 0, 0], k_weight=x[0, 0, 1]),
            fc.kv_cache_append: dict(key=x, value=x, key_cache=x, value_cache=x, lengths=torch.zeros(1, dtype=torch.int32)),
            fc.kv_cache_read: dict(key_cache=x, value_cache=x),
            fc.tree_attention: dict(query=x, key_cache=x, value_cache=x, lengths=torch.zeros(1, dtype=torch.int32))}[call]
    args = {n: t.clone() for n, t in args.items()}
    with torch.set_grad_enabled(grad):
        with forward_ad.dual_level():
            dual = {**args, name: _dual(args[name])}
            with pytest.raises(RuntimeError, match=f"{call.__name__} has no forward-mode derivative"):
                call(**dual)
            with pytest.raises(RuntimeError, match=f"{call.__name__} has no forward-mode derivative"):
                call(**{**dual, name: dual[name][:]})  # a view carries its base's tangent
            with pytest.raises(ValueError, match="CUDA device"):  # without tangents: the usual refusal of these CPU tensors
                call(**{**dual, name: forward_ad.unpack_dual(dual[name]).primal})
        with pytest.raises(ValueError, match="CUDA device"):
            call(**dual)  # the level is gone, and the tangents with it


def test_tangents_of_functional_transforms_are_refused():
    x = torch.zeros(1, 2, 3, 16, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="kv_cache_read has no forward-mode derivative"):
        torch.func.jvp(lambda k: fc.kv_cache_read(k, x)[0], (x,), (x,))


@pytest.mark.parametrize("scale", [3e38, -2.4e38])
def test_a_scale_that_overflows_in_base_2_is_refused(scale):
    """The kernels multiply by scale * log2(e): an infinite factor would turn scores of 0 into NaN."""
    x = torch.zeros(1, 2, 3, 16, dtype=torch.float16)
    with pytest.raises(ValueError, match="scale"):
        fc.tree_attention(x, x, x.clone(), torch.zeros(1, dtype=torch.int32), scale=scale)
    cache = nat.KvCache(1, 2, 3, 16, nat.FCR_KV_16BIT, nat.FCR_F16, (96, 48, 16, 1), (96, 48, 16, 1), (0, 0, 0), (0, 0, 0))
    for s, fine in ((scale, False), (2.3e38, True), (-2.3e38, True)):
        tree = nat.Tree(2, 3, (96, 48, 16, 1), 32, (0, 0), s)
        assert (nat.lib.fcr_tree_workspace_bytes(C.byref(cache), C.byref(tree), 148) > 0) == fine
        assert fine or "scale" in nat.last_error()


BIG = 2 ** 30 + 1


def _wide(*shape, dtype=torch.float16):
    return torch.zeros((1,) * (len(shape) - 1) + (shape[-1] if len(shape) == 4 else 1,), dtype=dtype).expand(shape)


@pytest.mark.parametrize("call", [
    lambda: fc.qk_norm_rope(_wide(1, 1, BIG, 2), _wide(1, 1, BIG, 2), _wide(BIG, dtype=torch.int32), torch.zeros(1)),
    lambda: fc.qk_norm_rope(_wide(1, BIG, 1, 2), _wide(1, 1, 1, 2), torch.zeros(1, dtype=torch.int32), torch.zeros(1)),
    lambda: fc.qk_norm_rope(_wide(1, BIG // 2 + 1, 1, 2), _wide(1, BIG // 2 + 1, 1, 2), torch.zeros(1, dtype=torch.int32), torch.zeros(1)),
    lambda: fc.kv_cache_read(_wide(1, 1, 2 ** 32 + 5, 8), _wide(1, 1, 2 ** 32 + 5, 8)),
    lambda: fc.kv_cache_read(_wide(2 ** 20, 2 ** 11, 1, 8), _wide(2 ** 20, 2 ** 11, 1, 8)),
    lambda: fc.kv_cache_read(_wide(1, 1, 5, 8), _wide(1, 1, 5, 8), positions=_wide(1, 1, BIG, dtype=torch.int32)),
    lambda: fc.kv_cache_append(_wide(1, 1, BIG, 8), _wide(1, 1, BIG, 8), torch.zeros(1, 1, 5, 8, dtype=torch.float16),
                               torch.zeros(1, 1, 5, 8, dtype=torch.float16), torch.zeros(1, dtype=torch.int32)),
    lambda: fc.tree_attention(_wide(1, 2 ** 23, 256, 8), _wide(1, 1, 5, 8), _wide(1, 1, 5, 8), torch.zeros(1, dtype=torch.int32)),
    lambda: fc.tree_attention(_wide(1, 1, 1, 8), _wide(1, 1, BIG, 8), _wide(1, 1, BIG, 8), torch.zeros(1, dtype=torch.int32)),
])
def test_sizes_that_32_bits_do_not_hold_are_refused(call):
    """The kernels count rows in 32 bits: a longer cache was cut to what those hold."""
    with pytest.raises(ValueError, match=str(2 ** 30)):
        call()


def test_the_c_entries_refuse_sizes_that_32_bits_do_not_hold():
    p, st = C.c_void_p(4096), nat.strides4((1, 1, 1, 1))  # never dereferenced: every refusal comes before any device work

    def cache(b=1, h=1, n=5):
        return C.byref(nat.KvCache(b, h, n, 8, nat.FCR_KV_16BIT, nat.FCR_F16, (40, 40, 8, 1), (40, 40, 8, 1), (0, 0, 0), (0, 0, 0)))

    def tree(hq=1, m=1):
        return C.byref(nat.Tree(hq, m, (8, 8, 8, 1), 32, (0, 0), 0.1))

    for c, t in ((cache(n=BIG), tree()), (cache(b=2 ** 16, h=2 ** 15), tree(hq=2 ** 15)), (cache(), tree(hq=2 ** 23, m=256))):
        assert nat.lib.fcr_tree_workspace_bytes(c, t, 148) == 0 and str(2 ** 30) in nat.last_error()
        assert nat.lib.fcr_tree_attention(c, t, p, p, p, None, None, p, None, p, None, p, 1 << 40, None) == nat.FCR_ERR_UNSUPPORTED
    assert nat.lib.fcr_kv_append(cache(n=BIG), p, p, None, None, p, st, p, st, 1, p, None, 32, None) == nat.FCR_ERR_UNSUPPORTED
    assert nat.lib.fcr_kv_append(cache(), p, p, None, None, p, st, p, st, BIG, p, None, 32, None) == nat.FCR_ERR_UNSUPPORTED
    assert nat.lib.fcr_kv_read(cache(n=BIG), p, p, None, None, None, 64, 1, p, p, None) == nat.FCR_ERR_UNSUPPORTED
    assert nat.lib.fcr_kv_read(cache(), p, p, None, None, p, 64, BIG, p, p, None) == nat.FCR_ERR_UNSUPPORTED
    for sizes in ((1, 1, 1, BIG), (1, BIG, 0, 1), (1, BIG // 2 + 1, BIG // 2 + 1, 1)):
        r = nat.Rope(*sizes, 16, 16, (1, 1, 1, 1), (1, 1, 1, 1), nat.FCR_F16, nat.FCR_F16, 0, 32, (0, 1), 1e-6)
        assert nat.lib.fcr_qk_norm_rope(C.byref(r), *[p] * 8, None) == nat.FCR_ERR_UNSUPPORTED, sizes
