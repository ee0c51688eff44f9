"""Norms of queries and keys of each head and their rotation by position, in
one launch: what stands between a layer's projections and its KV append.  (The
reference leaves it to the model's own operators.)"""
from __future__ import annotations

import torch

from . import _lib


def rope_table(max_positions, rotary_dim, theta=10000.0, device="cuda", inv_freq=None):
    """fp32 [max_positions, rotary_dim]: for each position the cosines, then
    the sines, of rotary_dim / 2 angles position * theta^(-2i / rotary_dim) (or
    position * inv_freq[i], for scaled variants).  Angles and functions are in
    64 bits: in 32 an angle of position 100000 is off by up to 0.004."""
    if rotary_dim <= 0 or rotary_dim % 8:
        raise ValueError(f"rotary_dim {rotary_dim} must be a positive multiple of 8")
    if inv_freq is None:
        i = torch.arange(rotary_dim // 2, dtype=torch.float64, device=device)
        inv_freq = torch.pow(torch.tensor(float(theta), dtype=torch.float64, device=device), -2.0 * i / rotary_dim)
    inv_freq = torch.as_tensor(inv_freq, dtype=torch.float64, device=device)
    if inv_freq.shape != (rotary_dim // 2,):
        raise ValueError(f"inv_freq must be [{rotary_dim // 2}], got {tuple(inv_freq.shape)}")
    angle = torch.arange(max_positions, dtype=torch.float64, device=device)[:, None] * inv_freq
    return torch.cat((angle.cos(), angle.sin()), dim=1).float()


def norm_rope(q, k, positions, table, q_weight=None, k_weight=None, eps=1e-6, interleaved=False, out=None):
    """Queries and keys normed head by head and rotated by their positions.

    q [T, Hq, D], k [T, Hkv, D]: bf16, fp16 or fp32, of any strides with unit
    head_dim stride (views of one projection's output, say); D a multiple of 8
    up to 512.  positions: [T], int64 or int32.  table: rope_table's, fp32
    [max_positions, rotary_dim]; its first rotary_dim <= D elements of a head
    turn, in pairs (i, i + rotary_dim / 2) or, ``interleaved``, (2i, 2i + 1).
    q_weight / k_weight [D], of q's dtype or fp32: x * weight / sqrt(mean(x^2) +
    eps) first; None: no norm.  fp32 throughout, rounded once.  A position
    outside the table makes its token's rows NaN.

    Returns (q', k'): new contiguous tensors, or ``out``, a pair which may be
    (q, k) itself but must not overlap them otherwise.  (The ordinary call runs
    in kvhot_torch, the rest here.)
    """
    if out is None:
        done = _lib.native().norm_rope(q, k, positions, table, q_weight, k_weight, eps, bool(interleaved))
        if done is not None:
            return done
    if q.dim() != 3 or k.dim() != 3 or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2]:
        raise ValueError(f"q {tuple(q.shape)} / k {tuple(k.shape)} must be [T, Hq, D] and [T, Hkv, D]")
    t, hq, d = q.shape
    hkv = k.shape[1]
    if k.dtype != q.dtype:
        raise TypeError(f"dtype mismatch: q {q.dtype}, k {k.dtype}")
    dtype = _lib.dtype_code(q.dtype)
    dev = q.device
    if dev.type != "cuda" or k.device != dev or positions.device != dev or table.device != dev:
        raise ValueError("q, k, positions and the table must be on one GPU")
    if positions.shape != (t,):
        raise ValueError(f"positions must be [{t}], got {tuple(positions.shape)}")
    if positions.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"positions must be int64 or int32, got {positions.dtype}")
    if table.dim() != 2 or table.dtype != torch.float32 or not table.is_contiguous():
        raise ValueError("table must be a contiguous fp32 [max_positions, rotary_dim]")
    weights = [w for w in (q_weight, k_weight) if w is not None]
    for w in weights:
        if w.shape != (d,) or not w.is_contiguous() or w.device != dev:
            raise ValueError(f"weights must be contiguous [{d}] on {dev}")
        if w.dtype not in (torch.float32, q.dtype) or w.dtype != weights[0].dtype:
            raise TypeError(f"weights must both be fp32 or {q.dtype}, got {w.dtype}")
    if out is None:
        oq, ok = (torch.empty(x.shape, dtype=x.dtype, device=dev) for x in (q, k))
    else:
        oq, ok = out
        for x, o in ((q, oq), (k, ok)):
            if o.shape != x.shape or o.dtype != x.dtype or o.device != dev:
                raise ValueError("out must be tensors of the shapes, dtype and device of q and k")
            if o.numel() and o.data_ptr() == x.data_ptr() and o.stride() != x.stride():
                raise ValueError("an output that overlaps its input must be the same view")
    if t == 0:
        return oq, ok
    positions = positions.contiguous()
    with torch.cuda.device(dev):
        status = _lib.load().kvhot_norm_rope(
            q.data_ptr(), _lib.i64_array(q.stride()), k.data_ptr(), _lib.i64_array(k.stride()),
            oq.data_ptr(), _lib.i64_array(oq.stride()), ok.data_ptr(), _lib.i64_array(ok.stride()),
            q_weight.data_ptr() if q_weight is not None else None,
            k_weight.data_ptr() if k_weight is not None else None,
            _lib.dtype_code(weights[0].dtype) if weights else dtype, float(eps), table.data_ptr(), table.shape[0],
            table.shape[1], 1 if interleaved else 0, positions.data_ptr(), 1 if positions.dtype is torch.int64 else 0,
            t, hq, hkv, d, dtype, _lib.stream_handle(dev))
    _lib.check(status, "kvhot_norm_rope")
    return oq, ok
