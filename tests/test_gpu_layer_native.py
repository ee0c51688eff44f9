"""kvhot_torch's side of the layer's calls: it takes the ordinary ones, gives
the bits that the Python functions give, and leaves the others to them."""
import pytest
import torch

from conftest import sea_module
from test_gpu_4bit import BF16, FP16, Step, announce
from test_native_calls import _Counted

pytestmark = pytest.mark.gpu


class _Nothing:
    def __getattr__(self, name):
        return lambda *args: None


def calls(cuda, sea):
    step = Step(sea, cuda, [(1, 700, 699), (5, 300, 295), (40, 40, 0)], 8, 2, 64, FP16)
    k, v = torch.randn(2, 1, 2, 30, 64, device=cuda, dtype=FP16)
    slots = torch.arange(30, device=cuda)
    qkv = torch.randn(9, 12, 64, device=cuda, dtype=BF16)
    w = torch.ones(64, device=cuda, dtype=BF16)
    table, pos = sea.rope_table(50, 64), torch.arange(9, device=cuda)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731

    def tables():
        m = sea.build_block_tables(i32([[1, 0, 0], [2, 3, 0]]), i32([5, 20]), i32([20, 3]), i32([7, 8, 9]), 25, 20)
        assert list(m) == ["q_lens", "k_lens", "q_starts", "q_pos_offsets", "block_table", "block_table_row_stride",
                           "total_query", "max_q_len", "max_k_len", "slot_mapping", "positions", "blocks_taken"]
        return [x if isinstance(x, torch.Tensor) else torch.tensor(x) for x in m.values()]

    # attention first: the append changes the cache
    return {"attention4": lambda: step.call(sea), "norm_rope": lambda: sea.norm_rope(qkv[:, :8], qkv[:, 8:10], pos, table, w),
            "tables": tables, "append4": lambda: [step.cache.write(k, v, 0, slots), step.cache.kv_cache][1:],
            "read4": lambda: step.cache.read(0, slots)}


def test_the_same_bits(cuda, sea, monkeypatch):
    lib = sea_module("_lib")
    counted = _Counted(lib.native())
    todo = calls(cuda, sea)
    for which, f in todo.items():
        announce("python", which)
        monkeypatch.setattr(lib, "_NATIVE", _Nothing())
        want = [x.clone() for x in f()]
        announce("native", which)
        monkeypatch.setattr(lib, "_NATIVE", counted)
        before = counted.taken
        got = f()
        assert counted.taken == before + 1 and counted.names[-1] == which
        assert len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want)), which


def test_other_calls_are_left_alone(cuda, sea):
    n = sea_module("_lib").native()
    for f in (n.append4, n.read4, n.attention4, n.norm_rope, n.tables):
        assert f() is None and f(*[None] * 5) is None and f(*[None] * 7) is None and f(*[None] * 8) is None and f(*[None] * 9) is None
    cache = sea._PagedKVCache4Bit(sea.allocate_kv_cache_4bit(1, 3, 2, 64), 64)
    k, slots = torch.zeros(1, 2, 4, 64, device=cuda, dtype=BF16), torch.arange(4, device=cuda)
    pool, code = cache.kv_cache, cache._code
    assert n.append4(pool, 64, code, k, k, 0, slots) is True
    for bad in ((pool, 64, code, k.half(), k, 0, slots), (pool, 64, code, k, k[:, :1], 0, slots), (pool, 64, code, k, k, 1, slots),
                (pool, 64, code, k, k, 0, slots[:3]), (pool, 64, code, k, k, 0, slots.cpu()), (pool, 96, code, k, k, 0, slots),
                (pool.cpu(), 64, code, k, k, 0, slots), (pool, 64, code, k, k, 0, slots.float())):
        assert n.append4(*bad) is None
    assert n.read4(pool, 64, code, 0, slots[:0]) is None and n.read4(pool, 64, code, -1, slots) is None
    with pytest.raises(IndexError):
        cache.read(-1, slots)
    with pytest.raises(IndexError):
        cache.write(k, k, 1, slots)
    with pytest.raises(ValueError):
        cache.write(k, k, 0, slots[:3])
    odd = torch.arange(8, device=cuda)[::2]
    cache.write(k, k, 0, odd)  # not contiguous: the Python function makes it so
    assert cache.read(0, odd)[0].shape == (4, 2, 64)
