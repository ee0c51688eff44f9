"""The KV side of a layer with a cache held in 4 bits, as measurable cases.

Four operators, each as a serving engine calls it:

* ``rope``: the norms of queries and keys of each head and their rotation by
  position, between a layer's projections and its append;
* ``update``: the append of a step's K/V to a cache held in 4 bits, and the
  dense read of cached tokens back (the cache's ``update``);
* ``attention``: paged attention of one layer over that cache, decode rows,
  rows of drafted tokens and prompt chunks mixed;
* ``tables``: a step's block tables, starts, slots and positions built on the
  GPU from the lengths of its rows.

The cache in memory: one record of 17 * head_dim bytes for each (block of 16
tokens, kv head).  In a record, first K's codes, token by token (element 2b in
the low half of byte b), then V's codes, element pair by element pair (byte
16 p + t holds elements 2p and 2p + 1 of token t), then the scales of K
(group by group of 32 elements, token 4 a + b at 4 b + a) and V (group by
group, token by token).  A code is a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4,
6; a scale byte x stands for 2^(x - 127), 255 for NaN.

Row lengths come from the case itself (``lens`` seeds them), values and block
placement from the seed given to ``prepare``.
"""
import importlib
import math
import random

import torch

own = False

BLOCK = 16
GROUP = 32
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
# Scale bytes that the quantiser gives: half the smallest and six times the
# largest scale are finite normal (fp16: representable) values of the type.
SCALES = {"bf16": (2, 252), "fp16": (104, 140), "fp32": (2, 252)}
EPS = 1e-6

_DEFAULTS = dict(kind="attention", dtype="bf16", hq=32, hkv=8, d=128, tokens=0, rotary=128, interleaved=False, norm=True,
                 far=8192, decode_rows=0, decode_lo=0, decode_hi=0, chunks=0, chunk_lo=0, chunk_hi=0, prior_lo=0,
                 prior_hi=0, causal=True, context=False, spare=0, pad=0, lens=1)


def _case(**kw):
    return {**_DEFAULTS, **kw}


def listed():
    return [
        # One interactive user's decode step: one token's heads.  Latency.
        _case(name="rope_1token", kind="rope", tokens=1),
        # A decode batch of a model that rotates half of each head, by
        # neighbouring pairs, and has no norms.
        _case(name="rope_57rows_fp16", kind="rope", dtype="fp16", hq=16, hkv=4, d=256, tokens=57, rotary=128,
              interleaved=True, norm=False, far=32768, lens=2),
        # A whole 8192-token prompt's heads.
        _case(name="rope_prompt_8192", kind="rope", tokens=8192, lens=3),
        # A decode step of 64 conversations appends one token each, and reads
        # those back.  Latency.
        _case(name="update_64rows", kind="update", decode_rows=64, decode_lo=128, decode_hi=2048, lens=2),
        # The append of a loaded step, 56 decode tokens and eight 512-token
        # chunks, and the dense read of every key that the step's rows see.
        _case(name="update_mixed_8x512", kind="update", decode_rows=56, decode_lo=256, decode_hi=2048, chunks=8,
              chunk_lo=512, chunk_hi=512, prior_lo=0, prior_hi=4096, context=True, lens=3),
        # One interactive user: a single decode row.
        _case(name="attention_1row", decode_rows=1, decode_lo=1001, decode_hi=1001),
        # An ordinary decode batch: 64 conversations.
        _case(name="attention_64rows", decode_rows=64, decode_lo=128, decode_hi=2048, lens=2),
        # Long documents: 16 rows of 32k tokens.
        _case(name="attention_long_16rows", decode_rows=16, decode_lo=32768, decode_hi=32768),
        # A step that verifies four drafted tokens a row, in fp16, with three
        # query heads to a kv head.
        _case(name="attention_drafts_24rows", dtype="fp16", hq=24, hkv=8, chunks=24, chunk_lo=5, chunk_hi=5, prior_lo=100,
              prior_hi=6000, lens=4),
        # A loaded engine with chunked prefill: 8 chunks of 512 tokens on
        # contexts of up to 4096, beside 56 decode rows.
        _case(name="attention_mixed_8x512", decode_rows=56, decode_lo=256, decode_hi=2048, chunks=8, chunk_lo=512,
              chunk_hi=512, prior_lo=0, prior_hi=4096, lens=3),
        # The tables of a decode step of 64 conversations.  Latency.
        _case(name="tables_64rows", kind="tables", decode_rows=64, decode_lo=128, decode_hi=2048, spare=8, lens=2),
        # The tables of a large engine's step: 1000 decode rows and 24 chunks.
        _case(name="tables_1024rows", kind="tables", decode_rows=1000, decode_lo=16, decode_hi=8192, chunks=24,
              chunk_lo=64, chunk_hi=1024, prior_lo=0, prior_hi=4096, spare=100, pad=37, lens=5),
    ]


# Head counts and head_dim of the models an engine serves.
_SHAPES = [(32, 8, 128), (32, 8, 128), (32, 8, 128), (8, 8, 128), (16, 8, 128), (64, 8, 128), (32, 8, 64),
           (24, 8, 128), (16, 4, 256), (12, 4, 96), (12, 12, 64), (8, 2, 64)]
# Bounds of a drawn case: bytes of the cache and of the dense tensors, and
# attention operations (fp32 arithmetic runs at a sixteenth of the 16-bit rate).
_MAX_BYTES = 1 << 30
_MAX_FLOPS = 1.4e11


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        c = _draw(rng)
        w = work(c)
        limit = _MAX_FLOPS / 16 if c["dtype"] == "fp32" else _MAX_FLOPS
        if w["bytes"] <= _MAX_BYTES and w["flops"] <= limit:
            return c


def _draw(rng):
    hq, hkv, d = rng.choice(_SHAPES)
    c = _case(hq=hq, hkv=hkv, d=d, dtype=rng.choice(["bf16", "bf16", "bf16", "fp16", "fp16", "fp32"]),
              lens=rng.randrange(1, 1 << 20))
    kind = rng.choice(["rope"] * 3 + ["update"] * 3 + ["attention"] * 8 + ["tables"] * 2)
    c["kind"] = kind
    if kind == "rope":
        c.update(tokens=_log_int(rng, 1, 8192), rotary=rng.choice([d, d, d, d // 2]), interleaved=rng.random() < 0.3,
                 norm=rng.random() < 0.7, far=_log_int(rng, 512, 131072))
        return c
    mix = rng.choice(["decode"] * 3 + ["drafts"] * 2 + ["chunks"] * 2 + ["mixed"] * 2)
    if mix in ("decode", "mixed"):
        hi = _log_int(rng, 16, 32768 if kind == "attention" else 4096)
        lo = hi if rng.random() < 0.2 else max(1, int(hi * rng.uniform(0.05, 0.9)))
        c.update(decode_rows=_log_int(rng, 1, 1024 if kind == "tables" else 256), decode_lo=lo, decode_hi=hi)
    if mix == "drafts":
        prior = _log_int(rng, 16, 16384)
        c.update(chunks=_log_int(rng, 1, 64), chunk_lo=2, chunk_hi=rng.randint(2, 9), prior_lo=prior // 5, prior_hi=prior)
    if mix in ("chunks", "mixed"):
        hi = _log_int(rng, 1, 4096 if mix == "chunks" else 1024)
        prior = 0 if rng.random() < 0.3 else _log_int(rng, 16, 16384)
        c.update(chunks=1 if rng.random() < 0.5 else _log_int(rng, 1, 16), chunk_lo=max(1, int(hi * rng.uniform(0.2, 1.0))),
                 chunk_hi=hi, prior_lo=prior // 4, prior_hi=prior)
    if kind == "update":
        c["context"] = rng.random() < 0.5
    if kind == "tables":
        c.update(spare=rng.randint(0, 64), pad=rng.choice([0, 0, rng.randint(1, 300)]))
    if kind == "attention":
        c["causal"] = rng.random() < 0.85
    return c


# ------------------------------------------------------------------ lengths --

def _rows(c):
    """(query tokens, keys, keys before them) of every row."""
    rng = random.Random(c["lens"])
    rows = []
    for _ in range(c["decode_rows"]):
        k = rng.randint(c["decode_lo"], c["decode_hi"])
        rows.append((1, k, k - 1))
    for _ in range(c["chunks"]):
        q = rng.randint(c["chunk_lo"], c["chunk_hi"])
        p = rng.randint(c["prior_lo"], c["prior_hi"])
        rows.append((q, p + q, p))
    return rows


def _nblocks(k):
    return -(-k // BLOCK)


def work(case):
    c = {**_DEFAULTS, **case}
    es = 4 if c["dtype"] == "fp32" else 2
    dense = c["hkv"] * c["d"] * es             # bytes of one token's K
    held = c["hkv"] * 17 * c["d"] // 16        # bytes of one token's K and V in the cache
    if c["kind"] == "rope":
        n = c["tokens"] * (c["hq"] + c["hkv"]) * c["d"]
        return {"bytes": float(2 * n * es + c["tokens"] * (4 * c["rotary"] + 8)), "flops": float(8 * n)}
    rows = _rows(c)
    tokens = sum(q for q, _, _ in rows)
    keys = sum(k for _, k, _ in rows)
    if c["kind"] == "update":
        read = keys if c["context"] else tokens
        return {"bytes": float(tokens * (2 * dense + held + 8) + read * (2 * dense + held + 8)), "flops": 0.0}
    if c["kind"] == "tables":
        fresh = sum(_nblocks(k) - _nblocks(p) for _, k, p in rows)
        return {"bytes": float(16 * len(rows) + 8 * fresh + 16 * (tokens + c["pad"]) + 4 * sum(_nblocks(q) for q, _, _ in rows)),
                "flops": 0.0}
    nbytes = keys * held + tokens * c["hq"] * (2 * c["d"] * es + 4) + 4 * sum(_nblocks(k) for _, k, _ in rows)
    pairs = sum(q * p + q * (q + 1) // 2 if c["causal"] else q * k for q, k, p in rows)
    return {"bytes": float(nbytes), "flops": float(4 * c["hq"] * c["d"] * pairs)}


# ------------------------------------------------------- the cache in memory --

_MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _quantise(x, dtype):
    """x [..., D] -> (codes uint8 [..., D], scale bytes uint8 [..., D / 32])."""
    lo, hi = SCALES[dtype]
    g = x.float().unflatten(-1, (-1, GROUP))
    top = g.abs().amax(-1)
    bits = top.view(torch.int32)
    byte = ((bits >> 23) + ((bits & 0x7fffff) > 0x600000).int() - 2).clamp(lo, hi)
    y = g * torch.exp2(127.0 - byte.float())[..., None]  # a power of two: exact
    a = y.abs()
    code = torch.where(a < 2, torch.round(2 * a), torch.where(a < 4, torch.round(a) + 2, torch.round(0.5 * a) + 4))
    code = code.clamp(max=7).to(torch.uint8) | (torch.signbit(y).to(torch.uint8) << 3)
    bad = ~torch.isfinite(top)
    byte = torch.where(bad, torch.full_like(byte, 255), byte)
    return code.masked_fill(bad[..., None], 0).flatten(-2), byte.to(torch.uint8)


def _parts(pool, d):
    """Views of a layer's records [N, Hkv, 17 D]: K codes [N, Hkv, 16, D / 2], V
    codes [N, Hkv, D / 2, 16], K scales [N, Hkv, D / 32, 4, 4], V scales [N,
    Hkv, D / 32, 16]."""
    kc, vc, ks, vs = pool.split([8 * d, 8 * d, d // 2, d // 2], dim=-1)
    return (kc.unflatten(-1, (BLOCK, d // 2)), vc.unflatten(-1, (d // 2, BLOCK)),
            ks.unflatten(-1, (d // GROUP, 4, 4)), vs.unflatten(-1, (d // GROUP, BLOCK)))


def _store(pool, d, dtype, blocks, tokens, k, v):
    """Writes k, v [T, Hkv, D] to tokens [T] of blocks [T] of the records."""
    kc, vc, ks, vs = _parts(pool, d)
    code, byte = _quantise(k, dtype)
    kc[blocks, :, tokens] = code[..., 0::2] | (code[..., 1::2] << 4)
    ks[blocks, :, :, tokens % 4, tokens // 4] = byte
    code, byte = _quantise(v, dtype)
    vc[blocks, :, :, tokens] = code[..., 0::2] | (code[..., 1::2] << 4)
    vs[blocks, :, :, tokens] = byte


def _dense(pool, d, blocks):
    """K and V, fp32 [len(blocks) * 16, Hkv, D] each, of blocks of the records."""
    kc, vc, ks, vs = _parts(pool[blocks], d)
    magnitude = torch.tensor(_MAGNITUDES + tuple(-m for m in _MAGNITUDES), device=pool.device)
    out = []
    for code, byte in ((kc, ks.transpose(-1, -2).flatten(-2)), (vc.transpose(-1, -2), vs)):
        code = torch.stack((code & 15, code >> 4), dim=-1).flatten(-2)           # [n, Hkv, 16, D]
        scale = torch.exp2(byte.float() - 127.0).transpose(-1, -2)               # [n, Hkv, 16, D / 32]
        x = magnitude[code.int()].unflatten(-1, (-1, GROUP)) * scale[..., None]
        out.append(x.flatten(-2).transpose(1, 2).reshape(-1, code.shape[1], d))
    return out


# ------------------------------------------------------------------- inputs --

def _placed(c, rows, seed):
    """(block table of every row, blocks in the pool): scattered blocks, a
    quarter of the pool unused."""
    need = [_nblocks(k) for _, k, _ in rows]
    total = sum(need)
    n = max(4, -(-5 * total // 4))
    ids, at, out = random.Random(seed).sample(range(n), total), 0, []
    for m in need:
        out.append(ids[at:at + m])
        at += m
    return out, n


def _scheduled(sea, c, rows, tables):
    out = sea.SchedulerOutput()
    for i, ((q, k, p), t) in enumerate(zip(rows, tables)):
        rid = f"r{i}"
        if i < c["decode_rows"]:
            req = sea.Request(rid, [0] * (k - 1), output_token_ids=[0], phase=sea.RequestPhase.NEEDS_DECODE,
                              block_table=t, num_computed_tokens=k - 1)
        else:
            req = sea.Request(rid, [0] * k, phase=sea.RequestPhase.NEEDS_PREFILL, block_table=t, num_computed_tokens=p)
            out.prefill_chunk_sizes[rid] = q
        out.scheduled_requests.append(req)
    return out


class _State:
    pass


def _sea():
    return importlib.import_module("serving-engine_amd")


def _rope_inputs(c, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(c["lens"])
    t, d, dt = c["tokens"], c["d"], DTYPES[c["dtype"]]
    # one projection's output holds q, k and v side by side
    qkv = torch.randn(t, c["hq"] + 2 * c["hkv"], d, generator=gen, device="cuda").mul_(2.0).to(dt)
    q, k = qkv[:, :c["hq"]], qkv[:, c["hq"]:c["hq"] + c["hkv"]]
    wq, wk = (1.0 + 0.2 * torch.randn(2, d, generator=gen, device="cuda")).to(dt)
    first = rng.randrange(0, max(1, c["far"] - t)) if t > 512 else None
    pos = list(range(first, first + t)) if first is not None else [rng.randrange(c["far"]) for _ in range(t)]
    if first is not None:
        pos = [min(p, c["far"] - 1) for p in pos]
    # cosines and sines from angles in 64 bits
    freq = torch.tensor([1e4 ** (-2 * i / c["rotary"]) for i in range(c["rotary"] // 2)], dtype=torch.float64, device="cuda")
    angle = torch.arange(c["far"], dtype=torch.float64, device="cuda")[:, None] * freq
    table = torch.cat((angle.cos(), angle.sin()), dim=1).float()
    return q, k, wq if c["norm"] else None, wk if c["norm"] else None, torch.tensor(pos, device="cuda"), table


def _cache_inputs(c, seed):
    """(rows, tables, blocks in the pool, chunks of the pool's K/V, q, k, v of the step)."""
    rows = _rows(c)
    tables, n = _placed(c, rows, seed)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kw = dict(generator=gen, device="cuda", dtype=DTYPES[c["dtype"]])
    t = sum(q for q, _, _ in rows)
    q = torch.randn(t, c["hq"], c["d"], **kw)
    k, v = torch.randn(t, c["hkv"], c["d"], **kw), torch.randn(t, c["hkv"], c["d"], **kw)
    step = max(1, (1 << 25) // (BLOCK * c["hkv"] * c["d"]))

    def contents():
        for b in range(0, n, step):
            m = min(step, n - b)
            yield b, torch.randn(2, m * BLOCK, c["hkv"], c["d"], **kw)

    return rows, tables, n, contents, q, k, v


def _slots(rows, tables):
    return [t[j // BLOCK] * BLOCK + j % BLOCK for (q, k, p), t in zip(rows, tables) for j in range(p, k)]


def _read_slots(c, rows, tables):
    if not c["context"]:
        return _slots(rows, tables)
    return [t[j // BLOCK] * BLOCK + j % BLOCK for (_, k, _), t in zip(rows, tables) for j in range(k)]


def _table_inputs(c, seed):
    """(rows, table with the blocks that the rows hold, free blocks)."""
    rows = _rows(c)
    ids = random.Random(seed)
    width = max(_nblocks(k) for _, k, _ in rows)
    held = [_nblocks(p) for _, _, p in rows]
    fresh = sum(_nblocks(k) for _, k, _ in rows) - sum(held)
    perm = list(range(sum(held) + fresh + c["spare"]))
    ids.shuffle(perm)
    table, at = [], 0
    for m in held:
        table.append(perm[at:at + m] + [0] * (width - m))
        at += m
    return rows, torch.tensor(table, dtype=torch.int32), torch.tensor(perm[at:], dtype=torch.int32)


def prepare(case, seed):
    c = {**_DEFAULTS, **case}
    s = _State()
    s.case = c
    s.sea = _sea() if own else None
    if c["kind"] == "rope":
        s.q, s.k, s.wq, s.wk, s.positions, s.table = _rope_inputs(c, seed)
        return s
    if c["kind"] == "tables":
        rows, table, free = _table_inputs(c, seed)
        s.table, s.free = table.cuda(), free.cuda()
        s.prior = torch.tensor([p for _, _, p in rows], dtype=torch.int32, device="cuda")
        s.q_lens = torch.tensor([q for q, _, _ in rows], dtype=torch.int32, device="cuda")
        s.total = sum(q for q, _, _ in rows) + c["pad"]
        s.max_q = max(q for q, _, _ in rows)
        return s
    rows, tables, n, contents, s.q, k, v = _cache_inputs(c, seed)
    s.rows = rows
    s.pool = torch.zeros(1, n, 1, c["hkv"], 17 * c["d"], dtype=torch.uint8, device="cuda")
    rec = s.pool[0, :, 0]
    for b, (pk, pv) in contents():
        at = torch.arange(pk.shape[0], device="cuda")
        _store(rec, c["d"], c["dtype"], b + at // BLOCK, at % BLOCK, pk, pv)
    if c["kind"] == "update":
        # [T, heads, D] from the projections; a model hands them on as [1, heads, T, D]
        s.k, s.v = k.transpose(0, 1).unsqueeze(0), v.transpose(0, 1).unsqueeze(0)
        s.write = torch.tensor(_slots(rows, tables), device="cuda")
        s.read = torch.tensor(_read_slots(c, rows, tables), device="cuda")
    else:
        s.tables = [torch.tensor(t, device="cuda") for t in tables]
        s.scale = 1.0 / math.sqrt(c["d"])
    if own:
        sea = s.sea
        s.cache = sea._PagedKVCache4Bit(s.pool, c["d"], dtype=DTYPES[c["dtype"]])
        if c["kind"] == "attention":
            s.meta = sea.step_inputs(_scheduled(sea, c, rows, tables), "cuda", s.cache)[0]
            s.blocks = s.cache.blocks(0)
    return s


# ---------------------------------------------------------------- the passes --

def _rotate(x, cos, sin, interleaved):
    """x [T, H, r] rotated by the angles of cos, sin [T, 1, r / 2]."""
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    a, b = x.chunk(2, dim=-1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)


def _rope_plain(s, c):
    cos, sin = s.table[s.positions][:, None].chunk(2, dim=-1)
    out = []
    for x, w in ((s.q, s.wq), (s.k, s.wk)):
        y = x.float()
        if w is not None:
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * w.float()
        y = torch.cat((_rotate(y[..., :c["rotary"]], cos, sin, c["interleaved"]), y[..., c["rotary"]:]), dim=-1)
        out.append(y.to(x.dtype))
    return tuple(out)


def _update_plain(s, c):
    rec, d = s.pool[0, :, 0], c["d"]
    _store(rec, d, c["dtype"], s.write // BLOCK, s.write % BLOCK, s.k[0].transpose(0, 1), s.v[0].transpose(0, 1))
    out = ([], [])
    for at in s.read.split(1 << 14):
        kc, vc, ks, vs = _parts(rec, d)
        b, t = at // BLOCK, at % BLOCK
        magnitude = torch.tensor(_MAGNITUDES + tuple(-m for m in _MAGNITUDES), device=rec.device)
        for o, code, byte in ((out[0], kc[b, :, t], ks[b, :, :, t % 4, t // 4]), (out[1], vc[b, :, :, t], vs[b, :, :, t])):
            code = torch.stack((code & 15, code >> 4), dim=-1).flatten(-2)
            x = magnitude[code.int()].unflatten(-1, (-1, GROUP)) * torch.exp2(byte.float() - 127.0)[..., None]
            o.append(x.flatten(-2).to(s.k.dtype))
    return torch.cat(out[0]), torch.cat(out[1])


def _attention_plain(s, c):
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    g = hq // hkv
    o, lse, at = [], [], 0
    for (n, m, p), table in zip(s.rows, s.tables):
        k, v = (x[:m].transpose(0, 1).contiguous() for x in _dense(s.pool[0, :, 0], d, table))   # [Hkv, m, D]
        q = s.q[at:at + n].float().unflatten(1, (hkv, g)).permute(1, 2, 0, 3).reshape(hkv, g * n, d)
        kt = k.transpose(1, 2).contiguous()
        hidden = None
        if c["causal"]:
            hidden = torch.arange(m, device=q.device)[None] > p + torch.arange(n, device=q.device)[:, None]
            hidden = hidden.repeat(g, 1)
        for h in range(0, hkv, max(1, (1 << 28) // (g * n * m))):
            e = min(hkv, h + max(1, (1 << 28) // (g * n * m)))
            x = torch.matmul(q[h:e], kt[h:e]) * s.scale
            if hidden is not None:
                x = x.masked_fill(hidden, -math.inf)
            top = x.amax(-1, keepdim=True)
            x = torch.exp(x - top)
            total = x.sum(-1, keepdim=True)
            y = torch.matmul(x, v[h:e]) / total
            o.append(y.view(e - h, g, n, d).permute(2, 0, 1, 3).reshape(n, (e - h) * g, d))
            lse.append((top + torch.log(total)).view(e - h, g, n).permute(2, 0, 1).reshape(n, (e - h) * g))
        parts = -(-hkv // max(1, (1 << 28) // (g * n * m)))
        o[-parts:], lse[-parts:] = [torch.cat(o[-parts:], dim=1)], [torch.cat(lse[-parts:], dim=1)]
        at += n
    return torch.cat(o).to(s.q.dtype), torch.cat(lse)


def _tables_plain(s):
    prior, q = s.prior.long(), s.q_lens.long()
    k = prior + q
    held, need = (prior + BLOCK - 1) // BLOCK, (k + BLOCK - 1) // BLOCK
    fresh = need - held
    ends = fresh.cumsum(0)
    col = torch.arange(s.table.shape[1], device=prior.device)[None]
    new = (col >= held[:, None]) & (col < need[:, None])
    source = ((ends - fresh)[:, None] + col - held[:, None]).clamp(0, s.free.numel() - 1)
    table = torch.where(new, s.free[source], s.table)
    starts = q.cumsum(0) - q
    token = torch.arange(s.total, device=prior.device)
    row = (torch.searchsorted(starts + q, token, right=True)).clamp(max=prior.numel() - 1)
    live = token < q.sum()
    pos = torch.where(live, prior[row] + token - starts[row], 0)
    slots = torch.where(live, table[row, pos // BLOCK].long() * BLOCK + pos % BLOCK, -1)
    return table, k.int(), starts.int(), slots, pos, ends[-1:].int()


def run(state):
    s, c = state, state.case
    kind = c["kind"]
    if own:
        sea = s.sea
        if kind == "rope":
            return sea.norm_rope(s.q, s.k, s.positions, s.table, s.wq, s.wk, eps=EPS, interleaved=c["interleaved"])
        if kind == "update":
            return s.cache.update(s.k, s.v, 0, s.read, s.write)
        if kind == "attention":
            return sea.paged_flash_attention_4bit(s.q, s.blocks, s.meta, c["hq"], c["hkv"], s.scale, is_causal=c["causal"])
        meta = sea.build_block_tables(s.table, s.prior, s.q_lens, s.free, total_query=s.total, max_q_len=s.max_q)
        return (meta["block_table"], meta["k_lens"], meta["q_starts"], meta["slot_mapping"], meta["positions"],
                meta["blocks_taken"])
    if kind == "rope":
        return _rope_plain(s, c)
    if kind == "update":
        return _update_plain(s, c)
    if kind == "attention":
        return _attention_plain(s, c)
    return _tables_plain(s)


# -------------------------------------------------------------------- exact --

def _held64(x, dtype):
    """What the cache holds of x [..., D], in 64 bits, from the definition: of
    the values m * 2^e with m one of +-_MAGNITUDES the nearest (of two as near
    the one with the even code), e the smallest exponent that leaves no value
    of the group of 32 off by more than 2^e."""
    lo, hi = SCALES[dtype]
    y = x.double().unflatten(-1, (-1, GROUP))
    top = y.abs().amax(-1)
    _, e = torch.frexp(top)                      # top = f * 2^e, f in [0.5, 1)
    # the smallest power s with top <= 7 s: s = 2^(e - 3) holds up to 8 s > top
    e = torch.where(top > torch.ldexp(torch.full_like(top, 7.0), e - 3), e - 2, e - 3)
    e = torch.where(top == 0, torch.full_like(e, lo - 127), e).clamp(lo - 127, hi - 127)[..., None]
    y = torch.ldexp(y, -e)
    m = torch.tensor(_MAGNITUDES, dtype=torch.float64, device=x.device)
    mid = (m[1:] + m[:-1]) / 2
    # a value on a border goes to the even one of the two codes
    up = torch.bucketize(y.abs(), mid, right=True)
    down = torch.bucketize(y.abs(), mid, right=False)
    z = torch.where(up % 2 == 0, m[up], m[down])
    return torch.ldexp(torch.where(y < 0, -z, z), e).flatten(-2)


def _exact_rope(c, seed):
    q, k, wq, wk, pos, table = _rope_inputs(c, seed)
    half = c["rotary"] // 2
    out = []
    for x, w in ((q, wq), (k, wk)):
        y = x.double()
        if w is not None:
            y = y / torch.sqrt((y ** 2).sum(-1, keepdim=True) / c["d"] + EPS) * w.double()
        z = y.clone()
        turn = torch.complex(table[pos, :half].double(), table[pos, half:].double())[:, None]
        at = torch.arange(half, device=x.device)
        a, b = (2 * at, 2 * at + 1) if c["interleaved"] else (at, at + half)
        r = torch.complex(y[..., a], y[..., b]) * turn
        z[..., a], z[..., b] = r.real, r.imag
        out.append(z)
    return tuple(out)


def _exact_update(c, seed):
    rows, tables, n, contents, _, k, v = _cache_inputs(c, seed)
    read = torch.tensor(_read_slots(c, rows, tables), device="cuda")
    out = [torch.empty(read.numel(), c["hkv"], c["d"], dtype=torch.float64, device="cuda") for _ in range(2)]
    for b, vals in contents():
        mine = ((read >= b * BLOCK) & (read < b * BLOCK + vals.shape[1])).nonzero()[:, 0]
        for o, x in zip(out, vals):
            o[mine] = _held64(x[read[mine] - b * BLOCK], c["dtype"])
    fresh = torch.full((n * BLOCK,), -1, device="cuda")
    written = torch.tensor(_slots(rows, tables), device="cuda")
    fresh[written] = torch.arange(written.numel(), device="cuda")
    mine = (fresh[read] >= 0).nonzero()[:, 0]
    for o, x in zip(out, (k, v)):
        o[mine] = _held64(x[fresh[read[mine]]], c["dtype"])
    return tuple(out)


def _exact_attention(c, seed):
    rows, tables, n, contents, q, _, _ = _cache_inputs(c, seed)
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    g = hq // hkv
    held = torch.empty(2, n * BLOCK, hkv, d, dtype=torch.float32, device="cuda")  # a code and a power of two: exact
    for b, vals in contents():
        held[:, b * BLOCK:b * BLOCK + vals.shape[1]] = _held64(vals, c["dtype"]).float()
    o = torch.empty(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(q.shape[:2], dtype=torch.float64, device="cuda")
    at = 0
    for (ql, kl, p), t in zip(rows, tables):
        slot = (torch.tensor(t, device="cuda")[:, None] * BLOCK + torch.arange(BLOCK, device="cuda")).flatten()[:kl]
        for h in range(hkv):
            k, v = held[0, slot, h].double(), held[1, slot, h].double()
            for j in range(h * g, h * g + g):
                for i in range(0, ql, 2048):
                    e = min(ql, i + 2048)
                    x = q[at + i:at + e, j].double() @ k.t().contiguous() / math.sqrt(d)
                    if c["causal"] and ql > 1:
                        see = torch.arange(kl, device="cuda")[None] <= p + torch.arange(i, e, device="cuda")[:, None]
                        x = torch.where(see, x, -math.inf)
                    ls = torch.logsumexp(x, -1)
                    lse[at + i:at + e, j] = ls
                    o[at + i:at + e, j] = torch.exp(x - ls[:, None]) @ v
        at += ql
    return o, lse


def _exact_tables(c, seed):
    rows, table, free = _table_inputs(c, seed)
    table, free = table.tolist(), free.tolist()
    taken, starts, slots, positions = 0, [], [], []
    for row, (q, k, p) in zip(table, rows):
        starts.append(len(slots))
        for j in range(p, k):
            if j % BLOCK == 0:  # the first token of a block takes one
                row[j // BLOCK] = free[taken]
                taken += 1
            slots.append(row[j // BLOCK] * BLOCK + j % BLOCK)
            positions.append(j)
    slots, positions = slots + [-1] * c["pad"], positions + [0] * c["pad"]
    return tuple(torch.tensor(x, dtype=torch.float64, device="cuda")
                 for x in (table, [k for _, k, _ in rows], starts, slots, positions, [taken]))


def exact(case, seed):
    c = {**_DEFAULTS, **case}
    if c["kind"] == "rope":
        return _exact_rope(c, seed)
    if c["kind"] == "update":
        return _exact_update(c, seed)
    if c["kind"] == "tables":
        return _exact_tables(c, seed)
    return _exact_attention(c, seed)
