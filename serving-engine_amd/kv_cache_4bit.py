"""A KV cache held in 4 bits, beside the 16- and 32-bit pool of model_runner.py.

A value is a code of 4 bits (a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6) times
a power of two that 32 elements of a head share: 17 bytes for 32 elements, so
a pool holds 3.76 times the tokens of a 16-bit one, and decode attention reads
that much less.  ``_PagedKVCache4Bit`` has ``_PagedKVCache``'s methods, and
``hip_paged_attention_forward`` takes either, so a model's steps
(``forward_step``, ``sample_step``, ``DecodeStepGraph``) run on it unchanged.

The reference caches in the model's dtype only
(serving_engine/model_runner.py:11-45, 101-125).
"""
from __future__ import annotations

import numpy as np
import torch

from . import _lib
from .block import BLOCK_SIZE
from .paged_attention_kernel import _WORKSPACES, _attend_into, _check_meta, _host_max, _order_list, _workspace

HEAD_DIMS_4BIT = (64, 96, 128, 256)
RECORD_TOKENS = 16  # tokens of a record; a block holds block_size / 16 of them a kv head


def record_bytes_4bit(head_dim: int) -> int:
    """Bytes that the K and V of 16 tokens of a kv head take."""
    if head_dim not in HEAD_DIMS_4BIT:
        raise ValueError(f"head_dim {head_dim} has no 4-bit cache; one of {HEAD_DIMS_4BIT}")
    return 17 * head_dim


def allocate_kv_cache_4bit(num_layers, num_blocks, num_kv_heads, head_dim, device="cuda", block_size=BLOCK_SIZE):
    """Zero-filled pool [L, N, block_size / 16, Hkv, 17 * D] of bytes
    (allocate_kv_cache's, in 4 bits); block_size is a multiple of 16."""
    if block_size <= 0 or block_size % RECORD_TOKENS:
        raise ValueError(f"block_size {block_size} must be a multiple of {RECORD_TOKENS}")
    return torch.zeros(num_layers, num_blocks, block_size // RECORD_TOKENS, num_kv_heads, record_bytes_4bit(head_dim),
                       dtype=torch.uint8, device=device)


def num_blocks_for_memory_4bit(free_bytes, num_layers, num_kv_heads, head_dim, gpu_memory_utilization=0.9,
                               block_size=BLOCK_SIZE):
    """num_blocks_for_memory for a pool in 4 bits."""
    per_block = num_layers * (block_size // RECORD_TOKENS) * num_kv_heads * record_bytes_4bit(head_dim)
    return int(free_bytes * gpu_memory_utilization) // per_block


def _check_blocks(blocks, dims):
    """A layer's records [N, S, Hkv, 17 D] (dims 4) or a pool of them (dims 5)."""
    if blocks.dim() != dims or blocks.dtype != torch.uint8:
        raise ValueError("a 4-bit cache is a uint8 tensor [" + ("num_layers, " if dims == 5 else "") +
                         "num_blocks, block_size / 16, num_kv_heads, 17 * head_dim]")
    s, h, rec = blocks.shape[-3:]
    if rec % 17 or rec // 17 not in HEAD_DIMS_4BIT:
        raise ValueError(f"records of {rec} bytes; 17 * head_dim for a head_dim of {HEAD_DIMS_4BIT}")
    if blocks.stride()[-3:] != (h * rec, rec, 1) and blocks.numel():
        raise ValueError("a block's records must be contiguous")


class _PagedKVCache4Bit:
    """_PagedKVCache over a pool of allocate_kv_cache_4bit.  ``dtype`` is the
    model's: what write takes and update returns."""

    def __init__(self, kv_cache: torch.Tensor, head_dim: int, dtype: torch.dtype = torch.bfloat16):
        _check_blocks(kv_cache, 5)
        if kv_cache.shape[4] != record_bytes_4bit(head_dim):
            raise ValueError(f"records of {kv_cache.shape[4]} bytes do not hold head_dim {head_dim}")
        self._code = _lib.dtype_code(dtype)
        self.kv_cache = kv_cache
        self.num_kv_heads = kv_cache.shape[3]
        self.head_dim = head_dim
        self.dtype = dtype

    @property
    def num_blocks(self):
        return self.kv_cache.shape[1]

    @property
    def block_size(self):
        return self.kv_cache.shape[2] * RECORD_TOKENS

    def _layer(self, layer_idx):
        kv = self.kv_cache
        if not 0 <= layer_idx < kv.shape[0]:
            raise IndexError(f"layer {layer_idx} outside the pool's {kv.shape[0]} layers")
        return kv.data_ptr() + layer_idx * kv.stride(0)

    def _index(self, name, index, n=None):
        if index.dim() != 1 or (n is not None and index.shape[0] != n):
            raise ValueError(f"{name} must be [{'slots' if n is None else n}], got {tuple(index.shape)}")
        if index.dtype not in (torch.int64, torch.int32):
            raise TypeError(f"{name} must be int64 or int32, got {index.dtype}")
        if index.device != self.kv_cache.device or index.device.type != "cuda":
            raise ValueError(f"{name} is on {index.device}, the cache on {self.kv_cache.device}")
        return index.contiguous()

    def write(self, key_states, value_states, layer_idx, write_index):
        """_PagedKVCache.write: quantises key_states / value_states [1, Hkv, S, D]
        into their slots, K and V in one launch.  The scale of 32 elements is
        the smallest power of two s with max|x| <= 7 s, held to [2^-125, 2^125]
        ([2^-23, 2^13] in fp16); codes are the nearest, ties to the even one.
        Elements that share a scale with an infinity or a NaN become NaN.
        Slots outside the pool are skipped; those inside must be distinct.
        (The ordinary call runs in kvhot_torch, as those of read and
        paged_flash_attention_4bit do; the rest here.)"""
        if _lib.native().append4(self.kv_cache, self.head_dim, self._code, key_states, value_states, layer_idx,
                                 write_index):
            return
        shape = key_states.shape
        if len(shape) != 4 or shape[0] != 1 or value_states.shape != shape:
            raise ValueError(f"key {tuple(key_states.shape)} / value {tuple(value_states.shape)} must be [1, Hkv, S, D]")
        _, hkv, s, d = shape
        if hkv != self.num_kv_heads or d != self.head_dim:
            raise ValueError(f"key/value heads/dim {hkv}/{d} do not match the cache {self.num_kv_heads}/{self.head_dim}")
        if key_states.dtype != self.dtype or value_states.dtype != self.dtype:
            raise TypeError(f"key/value dtype {key_states.dtype}/{value_states.dtype} is not the cache's {self.dtype}")
        kv = self.kv_cache
        if key_states.device != kv.device or value_states.device != kv.device:
            raise ValueError("key, value and the cache must be on one GPU")
        write_index = self._index("write_index", write_index, s)
        base = self._layer(layer_idx)
        if s == 0:
            return
        ks, vs = key_states.stride(), value_states.stride()
        with torch.cuda.device(kv.device):
            status = _lib.load().kvhot_reshape_and_cache_4bit(
                key_states.data_ptr(), _lib.i64_array((ks[2], ks[1], ks[3])),
                value_states.data_ptr(), _lib.i64_array((vs[2], vs[1], vs[3])), base, kv.stride(1),
                write_index.data_ptr(), 1 if write_index.dtype is torch.int64 else 0, s, hkv, d, self.block_size,
                self.num_blocks, _lib.dtype_code(self.dtype), _lib.stream_handle(kv.device))
        _lib.check(status, "kvhot_reshape_and_cache_4bit")

    def read(self, layer_idx, read_index):
        """What the cache holds at slots read_index: K and V, each a dense
        [len(read_index), Hkv, D] of the cache's dtype (zeros for a slot outside
        the pool)."""
        out = _lib.native().read4(self.kv_cache, self.head_dim, self._code, layer_idx, read_index)
        if out is not None:
            return out
        read_index = self._index("read_index", read_index)
        base = self._layer(layer_idx)
        kv, n = self.kv_cache, read_index.shape[0]
        key, value = (torch.empty(n, self.num_kv_heads, self.head_dim, dtype=self.dtype, device=kv.device)
                      for _ in range(2))
        if n:
            with torch.cuda.device(kv.device):
                status = _lib.load().kvhot_read_cache_4bit(
                    base, kv.stride(1), read_index.data_ptr(), 1 if read_index.dtype is torch.int64 else 0, n,
                    self.num_kv_heads, self.head_dim, self.block_size, self.num_blocks, key.data_ptr(),
                    value.data_ptr(), 0, _lib.dtype_code(self.dtype), _lib.stream_handle(kv.device))
            _lib.check(status, "kvhot_read_cache_4bit")
        return key, value

    def update(self, key_states, value_states, layer_idx, read_index, write_index):
        """_PagedKVCache.update: write, then the dense K and V of read_index."""
        self.write(key_states, value_states, layer_idx, write_index)
        return self.read(layer_idx, read_index)

    def blocks(self, layer_idx):
        """This layer's records, [N, block_size / 16, Hkv, 17 * D]: what
        paged_flash_attention_4bit takes."""
        return self.kv_cache[layer_idx]

    def copy_blocks(self, src_block_ids, dst_block_ids, validate=True):
        """_PagedKVCache.copy_blocks: the blocks of every layer, bit for bit, in
        one launch."""
        from .model_runner import _checked_pairs

        kv = self.kv_cache
        src, dst = _checked_pairs(src_block_ids, dst_block_ids, self.num_blocks, validate, kv.device)
        if src is None:
            return
        # The launch copies two ranges a block and layer (K and V): the halves
        # of a block's records.
        half = kv.shape[2] * kv.shape[3] * kv.shape[4] // 2
        with torch.cuda.device(kv.device):
            status = _lib.load().kvhot_copy_blocks(
                kv.data_ptr(), kv.shape[0], kv.stride(0), half, kv.stride(1), half, self.num_blocks, src.data_ptr(),
                dst.data_ptr(), src.numel(), _lib.stream_handle(kv.device))
        _lib.check(status, "kvhot_copy_blocks")


def paged_flash_attention_4bit(q, kv_blocks, metadata, num_q_heads, num_kv_heads, scale, is_causal=True):
    """paged_flash_attention over a cache held in 4 bits.

    q: [total_query, num_q_heads, head_dim] (any strides with unit head_dim
    stride), bf16, fp16 or fp32; kv_blocks: [num_blocks, block_size / 16,
    num_kv_heads, 17 * head_dim], a layer of the pool
    (``_PagedKVCache4Bit.blocks``); metadata: the dict of
    build_paged_batch_metadata or build_block_tables (where the former's host
    copies hold long prompts, those are planned from them, block table included,
    once a step).  Returns (o, l) as paged_flash_attention does, the same bits on
    every call.  A NaN in the cache reaches the queries that see it and no other.
    A pool written in another dtype may hold values beyond fp16's range; with fp16
    queries those are infinite, and an infinite value may also reach queries of a
    long prompt that do not see it.
    """
    out = _lib.native().attention4(q, kv_blocks, metadata, num_q_heads, num_kv_heads, scale, bool(is_causal), _WORKSPACES,
                                   PROMPT_PAIRS)
    if out is not None:
        return out
    if q.dim() != 3:
        raise ValueError("expected q [T, Hq, D]")
    _check_blocks(kv_blocks, 4)
    total_query, hq, head_dim = q.shape
    if hq != num_q_heads:
        raise ValueError(f"q has {hq} heads, num_q_heads={num_q_heads}")
    if num_kv_heads <= 0 or num_q_heads % num_kv_heads:
        raise ValueError(f"num_q_heads={num_q_heads} is not a multiple of num_kv_heads={num_kv_heads}")
    num_blocks, spb, hkv, rec = kv_blocks.shape
    if hkv != num_kv_heads or rec != 17 * head_dim:
        raise ValueError(f"cache shape {tuple(kv_blocks.shape)} does not match Hkv={num_kv_heads}, D={head_dim}")
    device = q.device
    if device.type != "cuda" or kv_blocks.device != device:
        raise ValueError("q and kv_blocks must be on the same GPU")
    _lib.dtype_code(q.dtype)
    q_lens = metadata["q_lens"]
    num_rows = q_lens.shape[0]
    o = torch.empty_like(q)
    l = torch.empty((total_query, num_q_heads), dtype=torch.float32, device=device)
    if num_rows == 0 or total_query == 0:
        return o, l
    for name in ("q_lens", "k_lens", "q_starts", "q_pos_offsets"):
        _check_meta(name, metadata[name], device, num_rows)
    bt = metadata["block_table"]
    _check_meta("block_table", bt, device, num_rows)
    bt_stride = int(metadata.get("block_table_row_stride", bt.shape[1] if bt.dim() == 2 else 0))
    max_q = _host_max(metadata, "max_q_len", "q_lens")
    max_k = _host_max(metadata, "max_k_len", "k_lens")
    plan = _prompts(metadata, device, num_q_heads, num_kv_heads, head_dim, spb * RECORD_TOKENS, q.dtype)
    with torch.cuda.device(device):
        if plan is None:
            _attend(q, kv_blocks, metadata, q_lens, total_query, max_q, max_k, bt_stride, scale, is_causal, o, l)
        else:
            if plan.max_q:
                _attend(q, kv_blocks, metadata, plan.q_lens, plan.sum_q, plan.max_q, plan.max_k, bt_stride, scale, is_causal,
                        o, l)
            _attend_prompts(q, kv_blocks, metadata, plan, bt_stride, scale, is_causal, o, l)
    return o, l


def _attend(q, kv_blocks, metadata, q_lens, sum_q, max_q, max_k, bt_stride, scale, is_causal, o, l):
    """kvhot_paged_attention_4bit of the rows that have queries in q_lens."""
    lib, device = _lib.load(), q.device
    total_query, hq, head_dim = q.shape
    num_blocks, spb, hkv, _ = kv_blocks.shape
    num_rows, dtype, stream = q_lens.shape[0], _lib.dtype_code(q.dtype), _lib.stream_handle(device)
    need = lib.kvhot_paged_attention_4bit_workspace_bytes(num_rows, sum_q, max_q, max_k, hq, hkv, head_dim, dtype)
    if need < 0:
        _lib.check(int(need), "kvhot_paged_attention_4bit_workspace_bytes")
    ws = _workspace(device, stream, need)
    status = lib.kvhot_paged_attention_4bit(
        q.data_ptr(), _lib.i64_array(q.stride()), kv_blocks.data_ptr(), kv_blocks.stride(0),
        o.data_ptr(), _lib.i64_array(o.stride()), l.data_ptr(), _lib.i64_array(l.stride()),
        metadata["block_table"].data_ptr(), bt_stride, q_lens.data_ptr(), metadata["k_lens"].data_ptr(),
        metadata["q_starts"].data_ptr(), metadata["q_pos_offsets"].data_ptr(),
        num_rows, total_query, sum_q, max_q, max_k, hq, hkv, head_dim, spb * RECORD_TOKENS, num_blocks,
        float(scale), _lib.KVHOT_CAUSAL if is_causal else 0, dtype,
        ws.data_ptr() if ws is not None else None, ws.numel() if ws is not None else 0, stream)
    _lib.check(status, "kvhot_paged_attention_4bit")


class _Prompts:
    """What a step's calls know of its prompts (rows that are attended over dense
    copies of their keys), planned once: ``meta``, the metadata of those
    rows alone over a pool of their own keys' copies, block after block; ``slots``
    [16 * blocks], where those keys are (-1 behind a row's end); ``rows``, their
    rows in the step's block table; ``q_lens``, the step's with theirs 0, and the
    bounds of the rows that are left."""


# A row with so many (query, head) pairs a kv head has its keys converted again for
# every 32 of them; copied once instead, they serve the 16-bit pools' attention,
# which then takes less time a pair.  The copies, the NaN's launch and the calls
# from Python cost about 50 us more: worth it from PROMPT_FLOPS on, all such rows
# together (bf16, 32 / 8 heads of 128, us a call from the 4-bit cache and over
# copies: 8 rows of 128 queries on 2048 keys, 32 GFLOP, 57 / 77, of 256, 62 GFLOP,
# 103 / 92, of 512 186 / 149; 300 queries on 5000 keys, 24 GFLOP, 54 / 58; 16 / 4
# heads of 256: 82 / 82, 155 / 108, 81 / 66).  In fp32, where the 4-bit kernel
# multiplies in three bf16 parts and the other on the fp32 matrix cores, never:
# 8 rows of 256 queries at 8 / 2 heads of 64 38 / 127.  Nor with groups of more than
# PROMPT_GROUP heads, which the other kernels attend without matrix cores.
PROMPT_PAIRS = 512
PROMPT_GROUP = 16
PROMPT_FLOPS = 35e9
# Bytes that a call's copies may take.
PROMPT_BYTES = 8 << 30


def _prompts(metadata, device, hq, hkv, d, block_size, dtype):
    """The step's _Prompts, planned from the host copies of its lengths and kept in
    the metadata; None without host copies or prompts."""
    host_q, group = metadata.get("host_q_lens"), hq // hkv
    if (host_q is None or dtype == torch.float32 or group > PROMPT_GROUP
            or _host_max(metadata, "max_q_len", "q_lens") * group < PROMPT_PAIRS):
        return None
    key = ("prompts4", hq, hkv, d, block_size, _lib.dtype_code(dtype), str(device))
    cache = metadata.setdefault("_schedules", {})
    if key in cache:
        hit = cache[key]
        _order_list(metadata, key, hit, device)
        return None if hit is None else hit[1]
    if torch.cuda.is_current_stream_capturing():
        return None  # (as _schedule: a copy from here would be replayed)
    host_k, host_bt = metadata["host_k_lens"], metadata["host_block_table"]
    rows = np.flatnonzero((host_q.astype(np.int64) * group >= PROMPT_PAIRS) & (host_k > 0))
    q_lens, k_lens = host_q[rows].astype(np.float64), host_k[rows].astype(np.int64)
    flops = 4.0 * hq * d * float((q_lens * (k_lens - q_lens / 2)).sum())  # causal
    blocks = -(-k_lens // BLOCK_SIZE)
    if (flops < PROMPT_FLOPS or int(blocks.sum()) * BLOCK_SIZE * hkv * d * 4 > PROMPT_BYTES
            or not rows.size or k_lens.max() > host_bt.shape[1] * block_size):
        cache[key] = None
        return None
    n = len(rows)
    ends = np.cumsum(blocks)
    total, width = int(ends[-1]), int(blocks.max())
    table = np.zeros((n, width), dtype=np.int32)
    slots = np.full((total, BLOCK_SIZE), -1, dtype=np.int64)
    for i, row in enumerate(rows):
        first = int(ends[i] - blocks[i])
        table[i, :blocks[i]] = np.arange(first, ends[i])
        j = np.arange(k_lens[i])
        slots[first:ends[i]].reshape(-1)[:k_lens[i]] = (
            host_bt[row, j // block_size].astype(np.int64) * block_size + j % block_size)
    short = host_q.copy()
    short[rows] = 0
    left = np.flatnonzero(short > 0)
    per_row = [metadata["host_" + x][rows].astype(np.int32) for x in ("q_lens", "k_lens", "q_starts", "q_pos_offsets")]
    ints = [short.astype(np.int32), *per_row, rows.astype(np.int32), table.reshape(-1)]
    at = np.cumsum([0] + [x.size for x in ints])
    pad = int(at[-1]) % 2  # the slots are 8-byte values
    staged = torch.empty(int(at[-1]) + pad + 2 * slots.size, dtype=torch.int32, pin_memory=True)
    staged.numpy()[:at[-1]] = np.concatenate(ints)
    staged.numpy()[at[-1] + pad:] = slots.reshape(-1).view(np.int32)
    buf = staged.to(device, non_blocking=True)
    dev = [buf[a:b] for a, b in zip(at[:-1], at[1:])]
    p = _Prompts()
    p.q_lens, p.rows, p.slots = dev[0], dev[5], buf[at[-1] + pad:].view(torch.int64)
    p.blocks = total
    p.sum_q, p.max_q = int(short[left].sum()), int(short.max()) if left.size else 0
    p.max_k = int(host_k[left].max()) if left.size else 0
    p.meta = dict(zip(("q_lens", "k_lens", "q_starts", "q_pos_offsets"), dev[1:5]))
    p.meta.update(zip(("host_q_lens", "host_k_lens", "host_q_starts", "host_q_pos_offsets"), per_row))
    p.meta.update(block_table=dev[6].view(n, width), host_block_table=table, block_table_row_stride=width,
                  max_q_len=int(per_row[0].max()), max_k_len=int(k_lens.max()))
    stream = torch.cuda.current_stream(device)
    event = torch.cuda.Event()
    event.record(stream)
    metadata.setdefault("_schedule_streams", {})[key] = (event, {stream.cuda_stream})
    cache[key] = (buf, p)
    return p


def _attend_prompts(q, kv_blocks, metadata, p, bt_stride, scale, is_causal, o, l):
    """The prompts' attention: their keys as dense copies, once for all their
    queries, then the 16-bit pools' attention over those, then the NaN that the
    copies left out."""
    lib, device, dtype = _lib.load(), q.device, _lib.dtype_code(q.dtype)
    num_blocks, spb, hkv, rec = kv_blocks.shape
    total_query, hq, d = q.shape
    stream = _lib.stream_handle(device)
    flags = _lib.KVHOT_CAUSAL if is_causal else 0
    pool = torch.empty(p.blocks, hkv, 2, BLOCK_SIZE, d, dtype=q.dtype, device=device)
    k, v = pool.permute(2, 0, 3, 1, 4)  # [blocks, tokens, Hkv, D] each, kv-interleaved
    status = lib.kvhot_read_cache_4bit(
        kv_blocks.data_ptr(), kv_blocks.stride(0), p.slots.data_ptr(), 1, p.blocks * BLOCK_SIZE, hkv, d,
        spb * RECORD_TOKENS, num_blocks, pool.data_ptr(), None, 1, dtype, stream)
    _lib.check(status, "kvhot_read_cache_4bit")
    _attend_into(q, k, v, p.meta, hq, hkv, scale, is_causal, 0, flags, o, l)
    m = p.meta
    status = lib.kvhot_spread_nan_4bit(
        kv_blocks.data_ptr(), kv_blocks.stride(0), o.data_ptr(), _lib.i64_array(o.stride()), l.data_ptr(),
        _lib.i64_array(l.stride()), metadata["block_table"].data_ptr(), bt_stride, p.rows.data_ptr(),
        m["q_lens"].data_ptr(), m["k_lens"].data_ptr(), m["q_starts"].data_ptr(), m["q_pos_offsets"].data_ptr(),
        p.rows.shape[0], total_query, m["max_q_len"], m["max_k_len"], hq, hkv, d, spb * RECORD_TOKENS, num_blocks, flags,
        dtype, stream)
    _lib.check(status, "kvhot_spread_nan_4bit")
