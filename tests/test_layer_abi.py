"""include/kvhot_layer.h: what it declares is exported, what it refuses is
refused on the host, before any launch (no GPU here); and the Python side's
own checks."""
import ctypes
import os
import re

import numpy as np
import pytest
import torch

import layer_ref as ref
from conftest import ROOT, sea_module

EINVAL, EUNSUPPORTED, EWORKSPACE = -1, -2, -3


@pytest.fixture(scope="module")
def lib():
    return sea_module("_lib").load()


def strides(*s):
    return (ctypes.c_int64 * len(s))(*s)


def test_every_declared_symbol_is_exported(lib):
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "kvhot_layer.h")).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(kvhot_\w+)\s*\(", text)))
    assert names == sorted(sea_module("_lib").LAYER_SIGNATURES)
    for n in names:
        assert hasattr(lib, n)


# Pointers that are checked, never followed: every call below is refused on the host.
P = 1 << 20


def append_args(**kw):
    a = dict(key=P, ks=strides(512, 128, 1), value=P, vs=strides(512, 128, 1), cache=P, block=4 * 17 * 128, slots=P, i64=1,
             tokens=3, heads=4, d=128, bs=16, blocks=10, dtype=2, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(key=None), EINVAL), (dict(slots=None), EINVAL), (dict(cache=None), EINVAL), (dict(ks=strides(512, 128, 2)), EINVAL),
    (dict(dtype=7), EINVAL), (dict(tokens=-1), EINVAL), (dict(heads=0), EINVAL), (dict(d=80), EUNSUPPORTED),
    (dict(bs=8), EUNSUPPORTED), (dict(bs=24), EUNSUPPORTED), (dict(cache=P + 8), EINVAL), (dict(block=4 * 17 * 128 + 8), EINVAL),
    (dict(block=17 * 128), EINVAL), (dict(key=P + 1), EINVAL), (dict(blocks=-1), EINVAL), (dict(tokens=1 << 40), EUNSUPPORTED),
])
def test_append_refusals(lib, kw, code):
    assert lib.kvhot_reshape_and_cache_4bit(*append_args(**kw)) == code
    assert lib.kvhot_last_error()


def test_calls_without_work_are_taken(lib):
    assert lib.kvhot_reshape_and_cache_4bit(*append_args(tokens=0, key=None)) == 0
    assert lib.kvhot_reshape_and_cache_4bit(*append_args(blocks=0, cache=None)) == 0
    assert lib.kvhot_read_cache_4bit(P, 4 * 17 * 128, None, 1, 0, 4, 128, 16, 10, None, None, 0, 2, None) == 0
    assert lib.kvhot_paged_attention_4bit(*attention_args(rows=0)) == 0
    assert lib.kvhot_paged_attention_4bit(*attention_args(total=0, sum_q=0)) == 0
    assert lib.kvhot_paged_attention_4bit(*attention_args(sum_q=0)) == 0
    assert lib.kvhot_norm_rope(*rope_args(tokens=0)) == 0


@pytest.mark.parametrize("kw,code", [
    (dict(slots=None), EINVAL), (dict(key=None), EINVAL), (dict(key=P + 4), EINVAL), (dict(n=-1), EINVAL),
    (dict(d=32), EUNSUPPORTED), (dict(dtype=5), EINVAL), (dict(value=None), EINVAL), (dict(blocks_too=1), EINVAL),
])
def test_read_refusals(lib, kw, code):
    a = dict(cache=P, block=4 * 17 * 128, slots=P, i64=1, n=5, heads=4, d=128, bs=16, blocks=10, key=P, value=P, blocks_too=0, dtype=2, s=None)
    a.update(kw)
    assert lib.kvhot_read_cache_4bit(*a.values()) == code


def attention_args(**kw):
    a = dict(q=P, qs=strides(1024, 128, 1), cache=P, block=4 * 17 * 128, out=P, os=strides(1024, 128, 1), lse=P,
             ls=strides(8, 1), bt=P, bt_stride=40, q_lens=P, k_lens=P, q_starts=P, offs=P, rows=3, total=3, sum_q=3, max_q=1,
             max_k=600, hq=8, hkv=4, d=128, bs=16, blocks=10, scale=0.1, flags=1, dtype=2, ws=None, ws_bytes=0, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), EINVAL), (dict(out=None), EINVAL), (dict(bt=None), EINVAL), (dict(k_lens=None), EINVAL),
    (dict(ls=None), EINVAL), (dict(qs=strides(1024, 1, 8)), EINVAL), (dict(hq=7), EINVAL), (dict(flags=2), EINVAL),
    (dict(flags=9), EINVAL), (dict(d=112), EUNSUPPORTED), (dict(bs=20), EUNSUPPORTED), (dict(dtype=3), EINVAL),
    (dict(blocks=0), EINVAL), (dict(max_k=1 << 33), EUNSUPPORTED), (dict(cache=P + 1), EINVAL), (dict(bt_stride=-1), EINVAL),
    (dict(max_k=100000), EWORKSPACE), (dict(sum_q=4), EINVAL), (dict(sum_q=-1), EINVAL), (dict(max_k=100000, ws=P, ws_bytes=64), EWORKSPACE), (dict(rows=-1), EINVAL),
])
def test_attention_refusals(lib, kw, code):
    assert lib.kvhot_paged_attention_4bit(*attention_args(**kw)) == code
    assert lib.kvhot_last_error()


def test_attention_workspace(lib):
    f = lib.kvhot_paged_attention_4bit_workspace_bytes
    assert f(1, 1, 1, 100, 8, 2, 128, 2) == 0           # one piece
    assert f(1, 1, 1, 100000, 8, 2, 128, 2) > 0
    assert f(0, 0, 0, 0, 8, 2, 128, 2) == 0
    assert f(1, 1, 1, 100, 8, 3, 128, 2) == EINVAL
    assert f(1, 1, 1, 100, 8, 2, 100, 2) == EUNSUPPORTED
    assert f(-1, 1, 1, 100, 8, 2, 128, 2) == EINVAL


def rope_args(**kw):
    a = dict(q=P, qs=strides(1024, 128, 1), k=P, ks=strides(512, 128, 1), qo=P, qos=strides(1024, 128, 1), ko=P,
             kos=strides(512, 128, 1), wq=P, wk=P, wdtype=2, eps=1e-6, table=P, rows=100, rotary=128, inter=0, pos=P, i64=1,
             tokens=3, hq=8, hkv=4, d=128, dtype=2, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), EINVAL), (dict(ko=None), EINVAL), (dict(pos=None), EINVAL), (dict(table=None), EINVAL),
    (dict(table=P + 4), EINVAL), (dict(rotary=136), EINVAL), (dict(rotary=4), EUNSUPPORTED), (dict(d=12, rotary=8), EUNSUPPORTED),
    (dict(d=520), EUNSUPPORTED), (dict(wdtype=1), EINVAL), (dict(wq=P + 1), EINVAL), (dict(qs=strides(1, 128, 8)), EINVAL),
    (dict(dtype=4), EINVAL), (dict(tokens=-1), EINVAL), (dict(q=P + 1), EINVAL),
])
def test_rope_refusals(lib, kw, code):
    assert lib.kvhot_norm_rope(*rope_args(**kw)) == code
    assert lib.kvhot_last_error()


@pytest.mark.parametrize("kw,code", [
    (dict(rows=0), EINVAL), (dict(rows=-1), EINVAL), (dict(bt=None), EINVAL), (dict(prior=None), EINVAL), (dict(free=None), EINVAL),
    (dict(slots=None), EINVAL), (dict(taken=None), EINVAL), (dict(bs=0), EINVAL), (dict(total=1 << 32), EUNSUPPORTED),
])
def test_table_refusals(lib, kw, code):
    a = dict(bt=P, stride=10, prior=P, q=P, free=P, n_free=5, rows=3, total=7, max_q=3, bs=16, starts=P, k=P, slots=P, pos=P,
             taken=P, stream=None)
    a.update(kw)
    assert lib.kvhot_build_block_tables(*a.values()) == code


def test_python_checks(sea):
    pool = sea.allocate_kv_cache_4bit(2, 5, 3, 96, device="cpu")
    assert pool.shape == (2, 5, 1, 3, 17 * 96)
    assert sea.allocate_kv_cache_4bit(1, 2, 1, 64, device="cpu", block_size=48).shape == (1, 2, 3, 1, 17 * 64)
    with pytest.raises(ValueError, match="multiple of 16"):
        sea.allocate_kv_cache_4bit(1, 2, 1, 64, device="cpu", block_size=24)
    with pytest.raises(ValueError, match="head_dim 80"):
        sea.allocate_kv_cache_4bit(1, 2, 1, 80, device="cpu")
    assert sea.num_blocks_for_memory_4bit(1 << 30, 2, 8, 128, 1.0) == (1 << 30) // (2 * 8 * 17 * 128)
    cache = sea._PagedKVCache4Bit(pool, 96)
    assert (cache.num_blocks, cache.block_size, cache.num_kv_heads) == (5, 16, 3)
    for bad, d, err in ((pool[0], 96, ValueError), (pool.float(), 96, ValueError), (pool, 64, ValueError),
                        (pool[..., :-1], 96, ValueError), (pool.transpose(2, 3), 96, ValueError)):
        with pytest.raises(err):
            sea._PagedKVCache4Bit(bad, d)
    with pytest.raises(TypeError):
        sea._PagedKVCache4Bit(pool, 96, dtype=torch.float64)
    k = torch.zeros(1, 3, 4, 96, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="is on cpu"):
        cache.write(k, k, 0, torch.zeros(4, dtype=torch.int64))
    with pytest.raises(TypeError):
        cache.write(k.half(), k.half(), 0, torch.zeros(4, dtype=torch.int64))
    with pytest.raises(ValueError):
        cache.write(k[:, :2], k[:, :2], 0, torch.zeros(4, dtype=torch.int64))
    with pytest.raises(ValueError, match="same GPU"):
        sea.paged_flash_attention_4bit(torch.zeros(1, 6, 96), cache.blocks(0), {}, 6, 3, 0.1)
    with pytest.raises(ValueError, match="does not match"):
        sea.paged_flash_attention_4bit(torch.zeros(1, 6, 64), cache.blocks(0), {}, 6, 3, 0.1)
    with pytest.raises(ValueError):
        sea.paged_flash_attention_4bit(torch.zeros(1, 6, 96), torch.zeros(5, 16, 3, 96), {}, 6, 3, 0.1)
    with pytest.raises(IndexError):
        cache.copy_blocks([0], [5])
    with pytest.raises(ValueError, match="unique"):
        cache.copy_blocks([0, 1], [2, 2])
    q, k = torch.zeros(2, 4, 64), torch.zeros(2, 2, 64)
    table = sea.rope_table(10, 64, device="cpu")
    with pytest.raises(ValueError, match="one GPU"):
        sea.norm_rope(q, k, torch.zeros(2, dtype=torch.int64), table)
    with pytest.raises(TypeError):
        sea.norm_rope(q, k.half(), torch.zeros(2, dtype=torch.int64), table)
    with pytest.raises(ValueError):
        sea.rope_table(10, 12, device="cpu")
    with pytest.raises(ValueError, match="GPU"):
        sea.build_block_tables(torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32),
                               torch.zeros(2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), 2, 1)


def test_rope_table_is_rounded_from_64_bits(sea):
    t = sea.rope_table(131072, 32, theta=5e5, device="cpu")
    assert t.shape == (131072, 32) and t.dtype == torch.float32
    for p in (0, 1, 131071):
        a = p * 5e5 ** (-2.0 * np.arange(16) / 32)
        want = np.concatenate((np.cos(a), np.sin(a)))
        # a rounding to fp32, and the 64-bit angle's own (131071 * 2^-52)
        assert (np.abs(t[p].numpy() - want) <= 2.0 ** -24 * np.abs(want) + 1e-9).all()


def test_reference_quantiser():
    """The oracle against the definition, value by value."""
    rng = np.random.default_rng(0)
    for dtype in ("bfloat16", "float16"):
        lo, hi = ref.SCALE_EXPONENTS[dtype]
        for scale in (1e-6, 1.0, 3e4):
            x = (rng.standard_normal((50, 32)) * scale)
            codes, bytes_ = ref.quantise(x, dtype)
            y = ref.values(codes, bytes_)
            s = np.ldexp(1.0, bytes_.astype(int) - 127)
            inside = np.abs(x).max(-1) <= 7 * s[:, 0]
            assert (np.abs(y - x) <= s)[inside].all()
            free = (bytes_[:, 0] > lo + 127) & inside
            assert (np.abs(x).max(-1) > 3.5 * s[:, 0])[free].all()  # no smaller scale would do
    codes, bytes_ = ref.quantise(np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, -0.25] + [6.0] * 24)[None], "bfloat16")
    assert bytes_[0, 0] == 127 and list(codes[0, :8]) == [0, 2, 2, 4, 4, 6, 6, 8]
    assert ref.quantise(np.array([7.0] + [0] * 31)[None], "bfloat16")[1][0, 0] == 127
    assert ref.quantise(np.array([7.0625] + [0] * 31)[None], "bfloat16")[1][0, 0] == 128
    assert ref.quantise(np.array([np.inf] + [0] * 31)[None], "bfloat16")[1][0, 0] == 255


@pytest.mark.parametrize("kw", [dict(rows=1 << 30), dict(total=1 << 31), dict(total=1 << 62, sum_q=1 << 62), dict(max_q=1 << 31),
                                dict(hq=1 << 17, hkv=1 << 17)])
def test_attention_sizes_beyond_the_kernels(lib, kw):
    assert lib.kvhot_paged_attention_4bit(*attention_args(**kw)) == EUNSUPPORTED
    a = dict(rows=3, total=3, max_q=1, max_k=600, hq=8, hkv=4, d=128, dtype=2)
    a.update({k: v for k, v in kw.items() if k in a})
    assert lib.kvhot_paged_attention_4bit_workspace_bytes(*a.values()) == EUNSUPPORTED
