"""The cache held in 4 bits through the package's entry points, against
layer_ref's 64-bit restatement: bytes and values exactly, attention within a
bound derived below."""
import math

import numpy as np
import pytest
import torch

import layer_ref as ref
from conftest import sea_module

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
HALF_STEP = {BF16: 2.0 ** -8, FP16: 2.0 ** -11, FP32: 2.0 ** -24}


def announce(*what):
    print("case:", *what, flush=True)


def name(dtype):
    return str(dtype).split(".")[1]


def f64(t):
    return t.detach().double().cpu().numpy()


# ------------------------------------------------------------ append and read --

@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("hkv,d,bs,strided,int32", [
    (3, 64, 16, False, False), (2, 96, 32, True, True), (8, 128, 16, True, False), (1, 256, 48, False, True),
    (2, 128, 64, False, False),
])
def test_append_writes_the_records_bytes(cuda, sea, dtype, hkv, d, bs, strided, int32):
    announce("append", dtype, hkv, d, bs, strided, int32)
    rng = np.random.default_rng(d + bs)
    n, layers, s = 7, 2, 37
    gen = torch.Generator(device="cuda").manual_seed(d)
    # rows of one projection: K and V beside other columns, token by token
    wide = torch.randn(s, 2 * hkv + 1, d, generator=gen, device=cuda)
    wide *= torch.exp2(torch.randint(-9, 9, (s, 2 * hkv + 1, 1), generator=gen, device=cuda))
    big, small = (3e4, 1e-7) if dtype is FP16 else (2e38, 1e-37)
    wide[0, :, :32], wide[1, :, 5], wide[2, :, :32] = 0, big, small
    wide[3, :, 7], wide[4, :, 40], wide[5, :, 0] = math.inf, math.nan, -math.inf
    wide[6, :, :8] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0], device=cuda)  # ties
    wide[6, :, 8:] = 0
    wide = wide.to(dtype)
    if strided and d != 96:
        wide = torch.cat((wide, wide[..., :1]), dim=-1)[..., :d]  # rows that start at odd elements
    k, v = wide[:, 1:1 + hkv], wide[:, 1 + hkv:]
    slots = rng.permutation(n * bs)[:s]
    slots[[8, 9]] = -1, n * bs
    slots[10] = np.iinfo(np.int32).max
    pool = torch.from_numpy(rng.integers(0, 255, (layers, n, bs // 16, hkv, 17 * d), dtype=np.uint8)).to(cuda)
    before = pool.cpu().numpy().copy()
    cache = sea._PagedKVCache4Bit(pool, d, dtype)
    index = torch.from_numpy(slots).to(cuda, torch.int32 if int32 else torch.int64)
    cache.write(k.transpose(0, 1).unsqueeze(0), v.transpose(0, 1).unsqueeze(0), 1, index)
    want = before.copy()
    kk, vv = f64(k), f64(v)
    for i, slot in enumerate(slots):
        if not 0 <= slot < n * bs:
            continue
        b, t = divmod(int(slot), bs)
        r, t = divmod(t, 16)
        for h in range(hkv):
            one = ref.record(np.repeat(kk[i, h][None], 16, 0), np.repeat(vv[i, h][None], 16, 0), name(dtype))
            w = want[1, b, r, h]
            w[t * d // 2:(t + 1) * d // 2] = one[t * d // 2:(t + 1) * d // 2]
            at = [8 * d + 16 * p + t for p in range(d // 2)]
            at += [16 * d + 16 * g + 4 * (t % 4) + t // 4 for g in range(d // 32)]
            at += [16 * d + d // 2 + 16 * g + t for g in range(d // 32)]
            w[at] = one[at]
    got = pool.cpu().numpy()
    assert np.array_equal(got[0], before[0])
    assert np.array_equal(got, want)
    # and back: what was written, exactly; zeros outside the pool
    announce("read", dtype, hkv, d, bs)
    rk, rv = cache.read(1, index)
    for x, y in ((rk, kk), (rv, vv)):
        held = ref.held(y, name(dtype))
        held[[8, 9, 10]] = 0
        assert np.array_equal(f64(x), held, equal_nan=True)


def test_update_reads_what_it_wrote(cuda, sea):
    cache = sea._PagedKVCache4Bit(sea.allocate_kv_cache_4bit(1, 9, 2, 64), 64, FP16)
    k, v = torch.randn(2, 1, 2, 20, 64, device=cuda, dtype=FP16)
    slots = torch.arange(40, 60, device=cuda)
    rk, rv = cache.update(k, v, 0, slots.flip(0), slots)
    for got, x in ((rk, k), (rv, v)):
        assert np.array_equal(f64(got)[::-1], ref.held(f64(x)[0].transpose(1, 0, 2), "float16"))
    empty = torch.zeros(0, dtype=torch.int64, device=cuda)
    assert cache.read(0, empty)[0].shape == (0, 2, 64)
    cache.write(k[:, :, :0], v[:, :, :0], 0, empty)


def test_copy_blocks(cuda, sea):
    pool = torch.randint(0, 255, (3, 12, 2, 3, 17 * 96), dtype=torch.uint8, device=cuda)
    want = pool.clone()
    want[:, [7, 2]] = want[:, [1, 11]]
    cache = sea._PagedKVCache4Bit(pool, 96)
    announce("copy of 4-bit blocks")
    cache.copy_blocks([1, 11], [7, 2])
    assert torch.equal(pool, want)
    cache.copy_blocks([], [])


# ------------------------------------------------------------------ attention --

class Step:
    """Rows (q_len, k_len, position of the first query) over a pool of scattered
    blocks; the values of every key come from the seed."""

    def __init__(self, sea, cuda, rows, hq, hkv, d, dtype, bs=16, seed=0, device_only=False, spare=3):
        rng = np.random.default_rng(seed)
        self.rows, self.hq, self.hkv, self.d, self.dtype = rows, hq, hkv, d, dtype
        need = [-(-k // bs) for _, k, _ in rows]
        n = sum(need) + spare
        ids = rng.permutation(n)
        width = max(max(need), 1) + 1
        table = rng.integers(0, 1 << 30, (len(rows), width)).astype(np.int32)  # garbage where nothing may read
        at = 0
        self.keys = []
        self.cache = sea._PagedKVCache4Bit(
            torch.randint(0, 255, (1, n, bs // 16, hkv, 17 * d), dtype=torch.uint8, device=cuda), d, dtype)
        for r, (_, k, _) in enumerate(rows):
            table[r, :need[r]] = ids[at:at + need[r]]
            at += need[r]
            kv = torch.from_numpy(rng.standard_normal((2, 1, hkv, k, d))).to(cuda, dtype)
            j = np.arange(k)
            slots = torch.from_numpy(table[r][j // bs].astype(np.int64) * bs + j % bs).to(cuda)
            self.cache.write(kv[0], kv[1], 0, slots)
            self.keys.append([ref.held(f64(x)[0].transpose(1, 0, 2), name(dtype)) for x in kv])
        q_lens = [q for q, _, _ in rows]
        starts = np.cumsum([0] + q_lens)
        self.total = int(starts[-1])
        self.starts = starts
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
        host = dict(q_lens=np.array(q_lens, np.int32), k_lens=np.array([k for _, k, _ in rows], np.int32),
                    q_starts=starts[:-1].astype(np.int32), q_pos_offsets=np.array([o for _, _, o in rows], np.int32))
        self.meta = {key: i32(x) for key, x in host.items()}
        self.meta.update(block_table=i32(table), block_table_row_stride=width, max_q_len=max(q_lens),
                         max_k_len=max(k for _, k, _ in rows), total_query=self.total)
        if not device_only:
            self.meta.update({"host_" + key: x for key, x in host.items()})
            self.meta["host_block_table"] = table
        self.q = torch.from_numpy(rng.standard_normal((max(self.total, 1), hq, d))).to(cuda, dtype)[:self.total]
        self.scale = 1.0 / math.sqrt(d)

    def call(self, sea, causal=True, q=None):
        return sea.paged_flash_attention_4bit(self.q if q is None else q, self.cache.blocks(0), self.meta, self.hq, self.hkv,
                                              self.scale, is_causal=causal)

    def expected(self, causal, q=None):
        q = f64(self.q if q is None else q)
        out = [ref.attention(q[s:s + n], k, v, off, self.scale, causal)
               for (n, _, off), s, (k, v) in zip(self.rows, self.starts, self.keys)]
        return [np.concatenate([x[i] for x in out]) for i in range(3)]

    def check(self, o, l, causal=True, q=None):
        """Bound of the error, from the arithmetic.  A score is a sum of D
        products in fp32 and its multiplication by the scale: off by e_s =
        (D + 4) 2^-24 sum|q k| scale, below that of the largest |q||k| here;
        exp2 and the running reference add 2^-20.  Each weight is thus off by e_s
        + 2^-20 relatively, and once more by its rounding to the type of the
        product (half a step; fp32: three bf16 parts, 2^-24); their sum likewise
        but for that rounding; sums of n terms add n 2^-24.  o = sum of weights
        times v, rounded to the type.  Relative to the largest, which the
        running reference keeps at 2^8 or above before the division, weights
        have a smallest step: 2^-126 of fp32's and bf16's normal numbers, 2^-24 of
        fp16's, so n weights lose up to n 2^-134 (n 2^-33) times max|v| whatever
        they sum to: an element whose large weights meet a v of 0 has no more than
        that of relative accuracy."""
        want, lse, bound = self.expected(causal, q)
        qn = np.linalg.norm(f64(self.q if q is None else q), axis=-1).max(initial=0)
        kn = max((np.linalg.norm(k, axis=-1).max() for k, _ in self.keys if k.size), default=0)
        kn = kn if np.isfinite(kn) else 100.0
        e_s = (self.d + 4) * 2.0 ** -24 * qn * kn * self.scale
        n = max(k for _, k, _ in self.rows)
        half = HALF_STEP[self.dtype]
        rel = half + 2 * (e_s + 2.0 ** -20 + n * 2.0 ** -24)
        got, gl = f64(o), f64(l)
        nan = np.isnan(want)
        assert np.array_equal(np.isnan(got), nan)
        fin = ~nan
        vmax = max((np.nanmax(np.abs(v), initial=0) for _, v in self.keys if v.size), default=0)
        # (with half of fp16's smallest step, in o itself)
        tiny = 2.0 ** -25 + n * 2.0 ** -33 * vmax if self.dtype is FP16 else n * 2.0 ** -134 * vmax
        err, tol = np.abs(got - want)[fin], (bound * rel + np.abs(want) * half + tiny)[fin]
        assert (err <= tol).all(), (err / np.maximum(tol, 1e-300)).max()
        assert np.array_equal(np.isnan(gl), np.isnan(lse))
        assert np.array_equal(np.isneginf(gl), np.isneginf(lse))
        fin = np.isfinite(lse)
        assert (np.abs(np.where(fin, gl, 0) - np.where(fin, lse, 0))[fin] <= e_s + 2.0 ** -20 + n * 2.0 ** -24 + 2.0 ** -23 * np.abs(lse[fin])).all()


SHAPES = [(8, 2, 128, BF16), (4, 4, 64, BF16), (6, 2, 96, FP16), (4, 1, 256, BF16), (12, 4, 64, FP16), (20, 1, 128, BF16),
          (16, 2, 128, FP16), (4, 2, 64, FP32), (6, 2, 96, FP32), (3, 1, 128, FP32), (2, 1, 256, FP32), (32, 1, 256, FP16)]
ROWS = {
    "decode": [(1, 1, 0), (1, 15, 14), (1, 16, 15), (1, 17, 16), (1, 64, 63), (1, 65, 64), (1, 257, 256), (1, 700, 699)],
    "drafts": [(5, 5, 0), (4, 131, 127), (2, 64, 62), (9, 1000, 991), (3, 66, 63)],
    "prompts": [(70, 70, 0), (33, 150, 117), (1, 2, 1), (129, 300, 171)],
    "odd": [(0, 40, 40), (2, 0, 0), (3, 20, -2), (1, 0, -1), (4, 30, 100), (0, 0, 0), (2, 35, 33)],
}


@pytest.mark.parametrize("hq,hkv,d,dtype", SHAPES)
@pytest.mark.parametrize("rows", list(ROWS))
def test_attention(cuda, sea, hq, hkv, d, dtype, rows):
    step = Step(sea, cuda, ROWS[rows], hq, hkv, d, dtype)
    for device_only in (False, True):
        if device_only:
            step.meta = {k: v for k, v in step.meta.items() if not k.startswith("host_")}
        for causal in (True, False):
            announce("attention", rows, hq, hkv, d, dtype, causal, device_only)
            o, l = step.call(sea, causal)
            step.check(o, l, causal)
            o2, l2 = step.call(sea, causal)
            assert torch.equal(o, o2) and torch.equal(l, l2)  # the same bits


@pytest.mark.parametrize("bs", [32, 48, 64])
def test_larger_blocks(cuda, sea, bs):
    step = Step(sea, cuda, ROWS["drafts"] + ROWS["decode"], 8, 2, 128, BF16, bs=bs)
    announce("blocks of", bs)
    step.check(*step.call(sea))


@pytest.mark.parametrize("rows", ["decode", "drafts", "prompts"])
def test_blocks_of_a_wider_pool(cuda, sea, rows):
    """Blocks with other bytes between them, layers too."""
    step = Step(sea, cuda, ROWS[rows], 8, 2, 128, BF16, bs=32)
    o, l = step.call(sea)
    pool = step.cache.kv_cache
    wide = torch.full((2, 2 * pool.shape[1], *pool.shape[2:]), 255, dtype=torch.uint8, device=cuda)  # NaN
    wide[1, ::2] = pool[0]
    step.cache = sea._PagedKVCache4Bit(wide[:, ::2], 128, BF16)
    announce("blocks of a wider pool", rows)
    o2, l2 = sea.paged_flash_attention_4bit(step.q, step.cache.blocks(1), step.meta, 8, 2, step.scale)
    assert torch.equal(o, o2) and torch.equal(l, l2)


@pytest.mark.parametrize("rows", ["decode", "drafts"])
def test_pages_outside_the_pool_stay_inside(cuda, sea, rows):
    """Block ids that no block has, in one row: the others' results are as they were."""
    step = Step(sea, cuda, ROWS[rows], 8, 2, 64, FP16)
    o, l = step.call(sea)
    bad = len(ROWS[rows]) - 2
    lo, hi = int(step.starts[bad]), int(step.starts[bad + 1])
    for page in (-1, step.cache.num_blocks, 2 ** 31 - 1, -2 ** 31):
        step.meta["block_table"][bad] = page
        announce("pages outside the pool", rows, page)
        o2, l2 = step.call(sea)
        for got, want in ((o2, o), (l2, l)):
            assert torch.equal(got[:lo], want[:lo]) and torch.equal(got[hi:], want[hi:])


@pytest.mark.parametrize("rows", [[(1, 20000, 19999)], [(3, 9001, 8998), (1, 33, 32)], [(300, 5000, 4700)],
                                  [(1, 4000 - 7 * i, 3999 - 7 * i) for i in range(40)] + [(200, 200, 0)]])
@pytest.mark.parametrize("hq,hkv,d,dtype", [(8, 2, 128, BF16), (2, 2, 64, FP16), (4, 1, 256, FP32)])
def test_long_rows_cut_into_parts(cuda, sea, rows, hq, hkv, d, dtype):
    step = Step(sea, cuda, rows, hq, hkv, d, dtype)
    announce("long rows", rows[0], hq, hkv, d, dtype)
    step.check(*step.call(sea))
    step.meta = {k: v for k, v in step.meta.items() if not k.startswith("host_")}
    announce("long rows, device metadata", rows[0], hq, hkv, d, dtype)
    step.check(*step.call(sea))


@pytest.mark.parametrize("hq,hkv,d,dtype", [(6, 2, 96, BF16), (4, 1, 64, FP16), (2, 2, 256, BF16), (20, 1, 128, FP16), (2, 1, 96, FP32)])
def test_long_rows_in_many_parts(cuda, sea, hq, hkv, d, dtype):
    """One row and a few of many parts; some without queries, short or seen in part."""
    for rows in ([(1, 33333, 33332)], [(2, 9000, 8990), (0, 7000, 7000), (1, 5, 4), (3, 20001, 19998)]):
        step = Step(sea, cuda, rows, hq, hkv, d, dtype)
        announce("many parts", rows, hq, hkv, d, dtype)
        for causal in (True, False):
            step.check(*step.call(sea, causal), causal)


def test_long_prompts_of_two_tiles_in_parts(cuda, sea):
    """A prompt of 1024 blocks of one tile on more keys than a block takes whole."""
    step = Step(sea, cuda, [(512, 8500, 7988)], 32, 2, 64, FP16, device_only=True)
    announce("two tiles in parts")
    step.check(*step.call(sea))


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_queries_of_any_strides(cuda, sea, dtype):
    step = Step(sea, cuda, ROWS["drafts"], 4, 2, 64, dtype)
    wide = torch.randn(step.total, 7, 65, device=cuda).to(dtype)
    for q in (wide[:, 1:5, :64], wide[:, 2:6, 1:], step.q.transpose(0, 1).contiguous().transpose(0, 1)):
        announce("strided queries", dtype, q.stride())
        o, l = step.call(sea, q=q)
        step.check(o, l, q=q)


@pytest.mark.parametrize("hq,hkv,d,dtype", [(8, 2, 128, BF16), (4, 2, 64, FP16), (6, 2, 96, BF16), (4, 1, 256, FP16), (2, 1, 128, FP32),
                                            (6, 2, 96, FP32)])
def test_nan_reaches_the_queries_that_see_it(cuda, sea, hq, hkv, d, dtype):
    """NaN in K and V: among the drafted tokens and prompts that see it in part,
    in the last block behind the row's end, at key 0."""
    rows = [(5, 40, 35), (1, 100, 99), (70, 133, 63), (1, 70, 69), (4, 64, 60), (40, 40, 0)]
    step = Step(sea, cuda, rows, hq, hkv, d, dtype)
    bad = [(0, 37, 1, 3), (0, 38, 0, 40), (1, 0, 1, d - 1), (2, 100, 1, 0), (2, 132, 0, 5), (3, 69, 0, 1), (4, 61, 1, 33),
           (5, 20, 1, 9), (5, 31, 0, 9)]  # row, key, K or V, element
    bt = step.meta["block_table"].cpu().numpy()
    for r, key, kv, el in bad:
        slot = torch.tensor([int(bt[r, key // 16]) * 16 + key % 16], device=cuda)
        now = [x.clone() for x in step.cache.read(0, slot)]
        now[kv][0, :, el] = math.nan
        step.cache.write(now[0].unsqueeze(0).transpose(1, 2), now[1].unsqueeze(0).transpose(1, 2), 0, slot)
        g = el // 32 * 32
        step.keys[r][kv][key, :, g:g + 32] = math.nan
    # (a value that was read back and appended again keeps its value)
    for causal in (True, False):
        announce("NaN", hq, hkv, d, dtype, causal)
        o, l = step.call(sea, causal)
        want, lse, _ = step.expected(causal)
        # numpy's product of a matrix adds 0 * NaN nowhere here: a query's keys are those it sees
        assert np.isnan(want).any() and not np.isnan(want).all()
        step.check(o, l, causal)


def test_extreme_scores(cuda, sea):
    """Scores that grow along the row, the largest last; all equal; very negative."""
    step = Step(sea, cuda, [(1, 400, 399), (6, 400, 394)], 4, 2, 64, BF16)
    for f in (30.0, -30.0, 0.0, 3000.0):
        q = (step.q.float() * f).to(BF16)
        announce("scores times", f)
        o, l = step.call(sea, q=q)
        step.check(o, l, q=q)


def test_other_scales(cuda, sea):
    """Negative (the largest scores are the smallest products) and zero (every key the same)."""
    step = Step(sea, cuda, [(1, 400, 399), (6, 70, 64), (40, 40, 0)], 4, 2, 64, FP16)
    for scale in (-0.3, 0.0):
        step.scale = scale
        announce("scale", scale)
        o, l = step.call(sea)
        step.scale = scale
        want, lse, bound = step.expected(True)
        assert (np.abs(f64(o) - want) <= 2.0 ** -9 * bound + 1e-6).all()
        assert (np.abs(f64(l) - lse) <= 1e-4).all()


def test_without_lse(cuda, sea):
    step = Step(sea, cuda, [(1, 3000, 2999), (3, 70, 67)], 4, 2, 64, BF16)
    lib = sea_module("_lib")
    want, _ = step.call(sea)
    m, c, q = step.meta, step.cache, step.q
    o = torch.zeros_like(q)
    need = lib.load().kvhot_paged_attention_4bit_workspace_bytes(2, 4, 3, 3000, 4, 2, 64, 2)
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device=cuda)
    announce("no lse")
    lib.check(lib.load().kvhot_paged_attention_4bit(
        q.data_ptr(), lib.i64_array(q.stride()), c.kv_cache.data_ptr(), c.kv_cache.stride(1), o.data_ptr(),
        lib.i64_array(o.stride()), None, None, m["block_table"].data_ptr(), m["block_table_row_stride"], m["q_lens"].data_ptr(),
        m["k_lens"].data_ptr(), m["q_starts"].data_ptr(), m["q_pos_offsets"].data_ptr(), 2, 4, 4, 3, 3000, 4, 2, 64, 16,
        c.num_blocks, step.scale, 1, 2, ws.data_ptr(), need, lib.stream_handle(cuda)), "kvhot_paged_attention_4bit")
    assert need > 0 and torch.equal(o, want)


@pytest.mark.parametrize("hq,hkv,d,dtype", [(32, 8, 128, BF16), (64, 8, 64, FP16)])
def test_many_rows_of_several_blocks(cuda, sea, hq, hkv, d, dtype):
    """More rows than a wave, some without queries, of one to many query blocks:
    the list of blocks on the device, one and two tiles a block."""
    rng = np.random.default_rng(1)
    for n, most in ((64, 30), (70, 3), (150, 12), (4200, 3)):
        rows = []
        for i in range(n):
            q = int(rng.integers(0, most)) if i % 5 else 0
            k = int(rng.integers(max(q, 1), 90 if n < 1000 else 12))
            rows.append((q, k, k - q))
        step = Step(sea, cuda, rows, hq, hkv, d, dtype)
        announce("many rows", n, most, hq, hkv, d, dtype)
        step.check(*step.call(sea))


@pytest.mark.parametrize("hq,hkv,d,dtype", [(16, 8, 128, BF16), (8, 8, 64, FP32)])
@pytest.mark.parametrize("n,most", [(95, 200), (96, 1024), (96, 1025), (191, 130), (192, 130)])
def test_many_short_rows(cuda, sea, hq, hkv, d, dtype, n, most):
    """Single tokens' rows around the numbers and lengths where a work-group has one,
    two and four waves; rows without keys and one that reaches the length."""
    rng = np.random.default_rng(2)
    lens = [most, 0, 1, 65] + [int(x) for x in rng.integers(0, most + 1, n - 4)]
    step = Step(sea, cuda, [(1, k, k - 1) for k in lens], hq, hkv, d, dtype)
    announce("many short rows", n, most, hq, hkv, d, dtype)
    o, l = step.call(sea)
    step.check(o, l)
    o2, l2 = step.call(sea)
    assert torch.equal(o, o2) and torch.equal(l, l2)


def test_pool_beyond_32_bits(cuda, sea):
    """Blocks whose bytes lie past 2^32 (17408 bytes a block)."""
    n = 300000
    pool = sea.allocate_kv_cache_4bit(1, n, 8, 128)
    cache = sea._PagedKVCache4Bit(pool, 128)
    blocks = [n - 1, 250001, 3, n - 2]
    keys = 61
    kv = torch.randn(2, 1, 8, keys, 128, device=cuda, dtype=BF16)
    slots = torch.tensor([blocks[j // 16] * 16 + j % 16 for j in range(keys)], device=cuda)
    announce("large pool")
    cache.write(kv[0], kv[1], 0, slots)
    rk, _ = cache.read(0, slots)
    held = [ref.held(f64(x)[0].transpose(1, 0, 2), "bfloat16") for x in kv]
    assert np.array_equal(f64(rk), held[0])
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    meta = dict(q_lens=i32(1), k_lens=i32(keys), q_starts=i32(0), q_pos_offsets=i32(keys - 1), block_table=i32(blocks),
                max_q_len=1, max_k_len=keys)
    q = torch.randn(1, 16, 128, device=cuda, dtype=BF16)
    o, l = sea.paged_flash_attention_4bit(q, cache.blocks(0), meta, 16, 8, 0.09)
    want, lse, bound = ref.attention(f64(q), held[0], held[1], keys - 1, 0.09, True)
    assert (np.abs(f64(o) - want) <= 2 * HALF_STEP[BF16] * bound + 1e-4 * bound).all()
    assert np.abs(f64(l) - lse).max() < 1e-4


# ------------------------------------------------------- streams and captures --

def test_streams_and_captures(cuda, sea):
    step = Step(sea, cuda, [(1, 5000, 4999), (5, 3000 - 900, 2095), (90, 500, 410)], 8, 2, 128, BF16)
    announce("eager")
    o, l = step.call(sea)
    torch.cuda.synchronize()
    step.check(o, l)
    outs = []
    for s in [torch.cuda.Stream() for _ in range(3)] * 2:
        with torch.cuda.stream(s):
            announce("on a stream")
            outs.append(step.call(sea))
    torch.cuda.synchronize()
    assert all(torch.equal(a, o) and torch.equal(b, l) for a, b in outs)
    graphs = []
    for fresh in (False, True):  # a step's later call, and its first one
        if fresh:
            step.meta = {k: v for k, v in step.meta.items() if not k.startswith("_")}
        g = torch.cuda.CUDAGraph()
        announce("capture", fresh)
        with torch.cuda.graph(g):
            out = step.call(sea)
        graphs.append((g, out))
    for _ in range(3):
        for g, out in graphs:
            out[0].zero_()
            out[1].zero_()
        for g, out in graphs:
            announce("replay")
            g.replay()
        step.call(sea)
        torch.cuda.synchronize()
        for g, out in graphs:
            step.check(*out)


def test_rows_beyond_the_last_query_are_left(cuda, sea):
    """Padded batches: queries that belong to no row keep their output."""
    step = Step(sea, cuda, [(1, 50, 49), (3, 20, 17)], 4, 2, 64, BF16)
    lib = sea_module("_lib")
    q = torch.cat((step.q, torch.randn(5, 4, 64, device=cuda, dtype=BF16)))
    o, l = torch.full_like(q, 7.0), torch.full((q.shape[0], 4), 7.0, device=cuda)
    m, c = step.meta, step.cache
    announce("padded batch")
    status = lib.load().kvhot_paged_attention_4bit(
        q.data_ptr(), lib.i64_array(q.stride()), c.kv_cache.data_ptr(), c.kv_cache.stride(1), o.data_ptr(),
        lib.i64_array(o.stride()), l.data_ptr(), lib.i64_array(l.stride()), m["block_table"].data_ptr(),
        m["block_table_row_stride"], m["q_lens"].data_ptr(), m["k_lens"].data_ptr(), m["q_starts"].data_ptr(),
        m["q_pos_offsets"].data_ptr(), 2, q.shape[0], 4, 3, 50, 4, 2, 64, 16, c.num_blocks, step.scale, 1, 2, None, 0,
        lib.stream_handle(cuda))
    lib.check(status, "kvhot_paged_attention_4bit")
    assert (o[4:] == 7).all() and (l[4:] == 7).all()
    step.check(o[:4], l[:4])


def test_lengths_beyond_their_bounds_stay_inside(cuda, sea):
    """Rows whose device lengths pass max_k_len or the table: the keys up to
    there are attended, nothing else is read."""
    step = Step(sea, cuda, [(1, 60, 59), (2, 60, 58)], 4, 2, 64, BF16)
    step.meta = {k: v for k, v in step.meta.items() if not k.startswith("host_")}
    step.meta["k_lens"].fill_(1 << 30)
    step.meta["q_pos_offsets"].fill_(1 << 30)
    step.meta["max_k_len"] = 60
    announce("lengths beyond max_k_len")
    o, l = step.call(sea)
    step.rows = [(1, 60, 59), (2, 60, 60)]
    step.check(o, l)


# ------------------------------------------------------------- as it is used --

def test_a_layer_of_a_step(cuda, sea):
    """Tables built on the device, norm and rotation, append, attention: two
    steps of a layer, the second of drafted tokens, against 64 bits on the
    values that the cache holds."""
    rng = np.random.default_rng(5)
    hq, hkv, d, bs, n = 8, 2, 64, 16, 40
    cache = sea._PagedKVCache4Bit(sea.allocate_kv_cache_4bit(1, n, hkv, d), d)
    table = sea.rope_table(256, d)
    w = (1 + 0.1 * torch.randn(d, device=cuda)).to(BF16)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    blocks, free = torch.zeros(3, 8, dtype=torch.int32, device=cuda), i32(rng.permutation(n).tolist())
    prior, taken = i32([0, 0, 0]), 0
    for q_lens in ([37, 5, 90], [3, 1, 5]):
        total = sum(q_lens) + 2
        meta = sea.build_block_tables(blocks, prior, i32(q_lens), free, total, max(q_lens))
        taken = int(meta["blocks_taken"])
        qkv = torch.randn(total, hq + 2 * hkv, d, device=cuda).to(BF16)
        q, k = sea.norm_rope(qkv[:, :hq], qkv[:, hq:hq + hkv], meta["positions"], table, w, w)
        v = qkv[:, hq + hkv:]

        class Layer:
            layer_idx = 0

        announce("layer", q_lens)
        o, _ = sea.hip_paged_attention_forward(
            Layer(), q.transpose(0, 1).unsqueeze(0), k.transpose(0, 1).unsqueeze(0), v.transpose(0, 1).unsqueeze(0), None,
            0.125, cache=cache, write_index=meta["slot_mapping"], paged_metadata=meta)
        bt, at = blocks.cpu().numpy(), 0
        for r, ql in enumerate(q_lens):
            p = int(prior[r])
            j = np.arange(p + ql)
            slots = torch.from_numpy(bt[r][j // bs].astype(np.int64) * bs + j % bs).to(cuda)
            kk, vv = (f64(x) for x in cache.read(0, slots))
            assert np.array_equal(kk[p:], ref.held(f64(k[at:at + ql]), "bfloat16"))
            want, _, bound = ref.attention(f64(q[at:at + ql]), kk, vv, p, 0.125, True)
            assert (np.abs(f64(o[0, at:at + ql]) - want) <= 2.1 * HALF_STEP[BF16] * bound).all()
            at += ql
        prior, free = meta["k_lens"].clone(), free[taken:].contiguous()


def test_engine_steps_on_a_4bit_cache(cuda, sea):
    """A whole model's steps (chunked prefill, decode, the recorded decode step)
    with the 4-bit cache in the place of the other."""
    transformers = pytest.importorskip("transformers")
    impl = sea.register_attention()
    cfg = transformers.LlamaConfig(hidden_size=256, intermediate_size=256, num_hidden_layers=2, num_attention_heads=4,
                                   num_key_value_heads=2, head_dim=64, vocab_size=97, attn_implementation=impl)
    torch.manual_seed(0)
    model = transformers.LlamaForCausalLM(cfg).to(cuda, BF16).eval()
    n = 64
    cache = sea._PagedKVCache4Bit(sea.allocate_kv_cache_4bit(2, n, 2, 64), 64)
    dense = sea._PagedKVCache(sea.allocate_kv_cache(2, n, 2, 64))
    tables = [list(range(5 * i, 5 * i + 5)) for i in range(2)]
    prompts = [list(range(1, 50)), list(range(3, 20))]
    logits = {}
    for kind, c in (("4bit", cache), ("16bit", dense)):
        out = sea.SchedulerOutput()
        for i, p in enumerate(prompts):
            out.scheduled_requests.append(sea.Request(f"r{i}", p, phase=sea.RequestPhase.NEEDS_PREFILL, block_table=tables[i],
                                                      num_computed_tokens=0))
            out.prefill_chunk_sizes[f"r{i}"] = len(p)
        announce("prefill step", kind)
        logits[kind] = sea.forward_step(model, out, c).float()
    # 4 bits of K and V against 16: the logits agree to the cache's error
    a, b = logits["4bit"], logits["16bit"]
    assert torch.isfinite(a).all()
    assert torch.nn.functional.cosine_similarity(a, b, dim=-1).min() > 0.9
    graph = sea.DecodeStepGraph(model, cache, 2, 8, 4, 2, 64, cuda)
    graph.tokens.copy_(logits["4bit"].argmax(-1))
    lens = [len(p) + 1 for p in prompts]
    for i in range(3):
        tokens = graph.tokens.clone()
        announce("recorded decode step", i)
        graph.step([x + i for x in lens], tables)
        got = graph.logits.float().clone()
        out = sea.SchedulerOutput()
        for j in range(2):
            out.scheduled_requests.append(sea.Request(
                f"r{j}", [0] * (lens[j] + i - 1), output_token_ids=[int(tokens[j])], phase=sea.RequestPhase.NEEDS_DECODE,
                block_table=tables[j], num_computed_tokens=lens[j] + i - 1))
        announce("eager decode step", i)
        eager = sea.forward_step(model, out, cache).float()
        # the same kernels on the same rows, planned for other bounds: bf16 roundings apart
        assert (got - eager).abs().max() <= 2 ** -5 * eager.abs().max()
