"""64-bit restatements, in numpy, of what include/kvhot_layer.h defines: the
4-bit quantiser and its bytes, attention, rotation, block tables.  Written from
the definitions alone."""
import numpy as np

MAGNITUDES = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=np.float64)
SCALE_EXPONENTS = {"bfloat16": (-125, 125), "float16": (-23, 13), "float32": (-125, 125)}


def quantise(x, dtype):
    """x [..., D] -> (codes [..., D], scale bytes [..., D / 32])."""
    lo, hi = SCALE_EXPONENTS[dtype]
    g = np.asarray(x, dtype=np.float64).reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    top = np.abs(g).max(-1, initial=0)
    good = np.isfinite(top)
    top, g = np.where(good, top, 0), np.where(good[..., None], g, 0)
    with np.errstate(divide="ignore"):
        e = np.maximum(np.floor(np.log2(top / 7)), lo - 1).astype(np.int64) - 1
    for _ in range(3):  # the smallest e with top <= 7 * 2^e
        e += np.ldexp(7.0, e) < top
    e = np.clip(e, lo, hi)
    a = np.abs(np.ldexp(g, -e[..., None]))
    codes = np.zeros(g.shape, dtype=np.uint8)
    near = np.full(g.shape, np.inf)
    for c in range(8):  # the nearest code; of two as near the even one
        dist = np.abs(a - MAGNITUDES[c])
        better = (dist < near) | ((dist == near) & (c % 2 == 0))
        codes, near = np.where(better, c, codes), np.where(better, dist, near)
    codes = np.where(good[..., None], codes | np.signbit(g) * 8, 0).astype(np.uint8)
    return codes.reshape(x.shape), np.where(good, e + 127, 255).astype(np.uint8)


def values(codes, scales):
    m = np.where(codes & 8, -1.0, 1.0) * MAGNITUDES[codes & 7]
    s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    return m * np.repeat(s, 32, axis=-1)


def held(x, dtype):
    """The values that the cache holds of x [..., D]."""
    return values(*quantise(x, dtype))


def record(k, v, dtype):
    """The 17 D bytes of 16 tokens' K and V [16, D], byte by byte as the header says."""
    d = k.shape[-1]
    out = np.zeros(17 * d, dtype=np.uint8)
    (kc, ks), (vc, vs) = quantise(k, dtype), quantise(v, dtype)
    for t in range(16):
        for b in range(d // 2):
            out[t * d // 2 + b] = kc[t, 2 * b] | kc[t, 2 * b + 1] << 4
            out[8 * d + 16 * b + t] = vc[t, 2 * b] | vc[t, 2 * b + 1] << 4
        for g in range(d // 32):
            out[16 * d + 16 * g + 4 * (t % 4) + t // 4] = ks[t, g]
            out[16 * d + d // 2 + 16 * g + t] = vs[t, g]
    return out


def attention(q, k, v, offset, scale, causal):
    """q [n, Hq, D] at positions offset.. over k, v [m, Hkv, D]: (o, lse, bound)
    with bound the sum of weight times |v|, the scale of o's error.  A query
    sums over the keys it sees and no others; none: o = 0, lse = -inf."""
    n, hq, d = q.shape
    m, hkv, _ = k.shape
    g = hq // hkv
    o, bound = np.zeros((n, hq, d)), np.zeros((n, hq, d))
    lse = np.full((n, hq), -np.inf)
    with np.errstate(all="ignore"):
        for i in range(n):
            c = m if not causal else min(m, max(0, offset + i + 1))
            if c == 0:
                continue
            s = np.matmul(q[i].reshape(hkv, g, d), k[:c].transpose(1, 2, 0)) * scale  # [Hkv, g, c]
            top = s.max(-1, keepdims=True)
            p = np.exp(s - top)
            total = p.sum(-1, keepdims=True)
            lse[i] = (top + np.log(total)).reshape(hq)
            p = p / total
            vv = v[:c].transpose(1, 0, 2)
            # (elementwise where a NaN is about: a product with a matrix adds 0 * NaN all the same)
            o[i] = np.matmul(p, vv).reshape(hq, d)
            bound[i] = np.matmul(p, np.abs(vv)).reshape(hq, d)
    return o, lse, bound


def norm_rope(x, weight, eps, cos, sin, interleaved):
    """x [T, H, D] with cos, sin [T, r / 2]: (y, scale of y's error)."""
    y = x.astype(np.float64)
    if weight is not None:
        y = y / np.sqrt((y ** 2).mean(-1, keepdims=True) + eps) * weight
    out, err = y.copy(), np.abs(y)
    half = cos.shape[1]
    for p in range(half):
        i, j = (2 * p, 2 * p + 1) if interleaved else (p, p + half)
        c, s = cos[:, None, p].astype(np.float64), sin[:, None, p].astype(np.float64)
        out[..., i] = y[..., i] * c - y[..., j] * s
        out[..., j] = y[..., j] * c + y[..., i] * s
        err[..., i] = err[..., j] = np.abs(y[..., i]) + np.abs(y[..., j])
    return out, err


def block_tables(table, prior, q_lens, free, total, bs):
    """(table, k_lens, q_starts, slots, positions, blocks taken), token by token."""
    table = [list(r) for r in table]
    taken, starts, slots, pos = 0, [], [], []
    for r, (p, q) in enumerate(zip(prior, q_lens)):
        p, q = max(p, 0), max(q, 0)
        starts.append(len(slots))
        for j in range(p, p + q):
            c = j // bs
            there = c < len(table[r])
            if j % bs == 0:
                there = there and taken < len(free)
                if c < len(table[r]):
                    table[r][c] = free[taken] if there else 0
                taken += 1
                fresh = there
            elif c * bs >= p:  # a block that this row took in this step
                there = fresh
            slots.append(table[r][c] * bs + j % bs if there else -1)
            pos.append(j)
    k_lens = [max(p, 0) + max(q, 0) for p, q in zip(prior, q_lens)]
    slots, pos = slots[:total], pos[:total]
    pad = total - len(slots)
    return table, k_lens, starts, slots + [-1] * pad, pos + [0] * pad, taken
