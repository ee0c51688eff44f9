"""norm_rope against 64 bits.  Bound of the error: the rounding to the type
(half a step) and fp32's: a sum of D squares is off by at most D 2^-24
relatively, its root by half of that, the divisions, root and products by 2^-24
each; a rotation adds three roundings of terms no larger than |a| + |b|."""
import numpy as np
import pytest
import torch

import layer_ref as ref

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
HALF_STEP = {BF16: 2.0 ** -8, FP16: 2.0 ** -11, FP32: 2.0 ** -24}


def f64(t):
    return t.detach().double().cpu().numpy()


def check(got, x, w, pos, table, interleaved, eps=1e-6):
    t = f64(table)[f64(pos).astype(np.int64)]
    half = table.shape[1] // 2
    want, scale = ref.norm_rope(f64(x), None if w is None else f64(w), eps, t[:, :half], t[:, half:], interleaved)
    h, d = HALF_STEP[x.dtype], x.shape[-1]
    tiny = 2.0 ** -25 if x.dtype is FP16 else 0.0
    tol = np.abs(want) * h * (1 + 2.0 ** -8) + scale * (d / 2 + 8) * 2.0 ** -24 + tiny
    assert (np.abs(f64(got) - want) <= tol).all()


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("d,rotary,interleaved,norm", [
    (128, 128, False, True), (128, 128, True, True), (64, 32, False, False), (96, 96, False, True), (256, 128, True, False),
    (80, 80, False, True), (8, 8, True, True), (512, 64, False, True), (200, 24, False, True), (72, 8, True, False),
])
@pytest.mark.parametrize("t,hq,hkv", [(1, 32, 8), (17, 6, 1), (300, 5, 5)])
def test_against_64_bits(cuda, sea, dtype, d, rotary, interleaved, norm, t, hq, hkv):
    print("case: norm_rope", dtype, d, rotary, interleaved, norm, t, hq, hkv, flush=True)
    gen = torch.Generator(device="cuda").manual_seed(t + d)
    qkv = (3 * torch.randn(t, hq + 2 * hkv, d, generator=gen, device=cuda)).to(dtype)
    q, k = qkv[:, :hq], qkv[:, hq:hq + hkv]
    w = (1 + 0.3 * torch.randn(2, d, generator=gen, device=cuda)).to(dtype) if norm else [None, None]
    pos = torch.randint(0, 5000, (t,), generator=gen, device=cuda)
    table = sea.rope_table(5000, rotary)
    oq, ok = sea.norm_rope(q, k, pos, table, w[0], w[1], interleaved=interleaved)
    assert oq.is_contiguous() and oq.shape == q.shape and ok.shape == k.shape
    check(oq, q, w[0], pos, table, interleaved)
    check(ok, k, w[1], pos, table, interleaved)
    # in place, int32 positions, the same bits
    a, b = sea.norm_rope(q, k, pos.int(), table, w[0], w[1], interleaved=interleaved, out=(q, k))
    assert a is q and torch.equal(q, oq) and torch.equal(k, ok)


@pytest.mark.parametrize("dtype,d,t", [(BF16, 128, 8192), (FP32, 64, 8195), (FP16, 256, 4100), (BF16, 512, 1700)])
def test_long_prompts(cuda, sea, dtype, d, t):
    """Outputs beyond 32 MiB take two sets of heads a wave: 21 heads, an odd count."""
    print("case: norm_rope long", dtype, d, t, flush=True)
    gen = torch.Generator(device="cuda").manual_seed(d)
    qkv = torch.randn(t, 21, d, generator=gen, device=cuda).to(dtype)
    w = (1 + 0.3 * torch.randn(2, d, generator=gen, device=cuda)).to(dtype)
    pos, table = torch.arange(t, device=cuda), sea.rope_table(t, d)
    oq, ok = sea.norm_rope(qkv[:, :17], qkv[:, 17:], pos, table, w[0], w[1])
    for s in (slice(0, 70), slice(t // 2, t // 2 + 70), slice(t - 70, t)):
        check(oq[s], qkv[s, :17], w[0], pos[s], table, False)
        check(ok[s], qkv[s, 17:], w[1], pos[s], table, False)
    # every row the same as in small calls, in place too
    parts = [sea.norm_rope(qkv[i:i + 500, :17], qkv[i:i + 500, 17:], pos[i:i + 500], table, w[0], w[1]) for i in range(0, t, 500)]
    assert torch.equal(oq, torch.cat([p[0] for p in parts])) and torch.equal(ok, torch.cat([p[1] for p in parts]))
    sea.norm_rope(qkv[:, :17], qkv[:, 17:], pos, table, w[0], w[1], out=(qkv[:, :17], qkv[:, 17:]))
    assert torch.equal(qkv[:, :17], oq) and torch.equal(qkv[:, 17:], ok)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_layouts_weights_and_no_heads(cuda, sea, dtype):
    table = sea.rope_table(64, 64)
    pos = torch.arange(9, device=cuda) * 7
    wide = torch.randn(9, 11, 131, device=cuda).to(dtype)
    head_major = torch.randn(4, 9, 64, device=cuda).to(dtype)
    w32 = 1 + 0.1 * torch.randn(65, device=cuda)
    for q, k in ((wide[:, 1:6, 1:65], wide[:, 6:9, 66:130]), (head_major.transpose(0, 1), wide[:, :1, :64]),
                 (wide[:, :0, :64], wide[:, 3:5, 64:128]), (wide[:, 3:5, 64:128], wide[:, :0, :64])):
        for wq, wk in ((w32[1:], None), (None, w32[:64]), (w32[:64].to(dtype), w32[1:].to(dtype))):
            print("case: norm_rope layout", dtype, q.stride(), k.stride(), flush=True)
            out = tuple(torch.zeros(9, x.shape[1], 67, device=cuda, dtype=dtype)[..., 2:66] for x in (q, k))
            oq, ok = sea.norm_rope(q, k, pos, table, wq, wk, eps=1e-3, out=out)
            check(oq, q, wq, pos, table, False, 1e-3)
            check(ok, k, wk, pos, table, False, 1e-3)


def test_positions_outside_the_table(cuda, sea):
    q, k = torch.randn(4, 2, 64, device=cuda), torch.randn(4, 1, 64, device=cuda)
    pos = torch.tensor([-1, 0, 9, 10], device=cuda)
    oq, ok = sea.norm_rope(q, k, pos, sea.rope_table(10, 32))
    for o in (oq, ok):
        assert torch.isnan(o[[0, 3]]).all() and torch.isfinite(o[[1, 2]]).all()


def test_zeros_infinities_and_nan_stay_in_their_head(cuda, sea):
    q = torch.randn(3, 4, 128, device=cuda, dtype=BF16)
    k = torch.randn(3, 2, 128, device=cuda, dtype=BF16)
    w = torch.ones(128, device=cuda, dtype=BF16)
    clean = sea.norm_rope(q, k, torch.arange(3, device=cuda), sea.rope_table(3, 128), w, w)
    q[0, 0], q[1, 1, 5], q[2, 2, 7], k[1, 0] = 0, float("inf"), float("nan"), 0
    oq, ok = sea.norm_rope(q, k, torch.arange(3, device=cuda), sea.rope_table(3, 128), w, w)
    assert (oq[0, 0] == 0).all() and (ok[1, 0] == 0).all()
    assert torch.isnan(oq[1, 1]).any() and torch.isnan(oq[2, 2]).all()
    keep = torch.ones(3, 4, dtype=torch.bool, device=cuda)
    keep[0, 0] = keep[1, 1] = keep[2, 2] = False
    assert torch.equal(oq[keep], clean[0][keep])


def test_empty_streams_and_captures(cuda, sea):
    table = sea.rope_table(100, 128)
    q, k = torch.randn(50, 8, 128, device=cuda, dtype=BF16), torch.randn(50, 2, 128, device=cuda, dtype=BF16)
    pos = torch.arange(50, device=cuda)
    assert sea.norm_rope(q[:0], k[:0], pos[:0], table)[0].shape == (0, 8, 128)
    want = sea.norm_rope(q, k, pos, table)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        other = sea.norm_rope(q, k, pos, table)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = sea.norm_rope(q, k, pos, table)
    for _ in range(3):
        out[0].zero_()
        g.replay()
        torch.cuda.synchronize()
        for o in (other, out):
            assert torch.equal(o[0], want[0]) and torch.equal(o[1], want[1])


def test_refusals(cuda, sea):
    table = sea.rope_table(10, 64)
    q, k, pos = torch.randn(2, 4, 64, device=cuda), torch.randn(2, 2, 64, device=cuda), torch.zeros(2, dtype=torch.int64, device=cuda)
    lib_error = RuntimeError
    for args, err in (((q, k[:1], pos, table), ValueError), ((q, k.half(), pos, table), TypeError),
                      ((q, k, pos[:1], table), ValueError), ((q, k, pos.float(), table), TypeError),
                      ((q, k, pos, table.half()), ValueError), ((q, k, pos, table, torch.ones(63, device=cuda)), ValueError),
                      ((q, k, pos, table, torch.ones(64, device=cuda, dtype=FP16)), TypeError),
                      ((q.transpose(1, 2).contiguous().transpose(1, 2), k, pos, table), lib_error),
                      ((q[..., :32], k[..., :32], pos, table), lib_error), ((q[..., :60], k[..., :60], pos, table), lib_error),
                      ((q.cpu(), k, pos, table), ValueError)):
        with pytest.raises(err):
            sea.norm_rope(*args)
    with pytest.raises(ValueError):
        sea.norm_rope(q, k, pos, table, out=(q[:, :, :32], k))
    with pytest.raises(ValueError, match="same view"):
        sea.norm_rope(q, k, pos, table, out=(q.as_strided(q.shape, (64, 128, 1)), k))
