"""Rows that the host knows to be prompts are attended over dense copies of their
keys: the same bound as the other rows', the same reach of a NaN, beside decode
rows, on other streams and in graphs."""
import math

import numpy as np
import pytest
import torch

from conftest import sea_module
from test_gpu_4bit import BF16, FP16, FP32, Step, announce, f64

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def small_prompts(monkeypatch):
    """Rows of these tests' sizes as prompts."""
    monkeypatch.setattr(sea_module("kv_cache_4bit"), "PROMPT_FLOPS", 0)


ROWS = [(1, 300, 299), (150, 400, 250), (3, 77, 74), (131, 131, 0), (1, 16, 15), (0, 9, 9), (200, 217, 17)]
SHAPES = [(8, 2, 128, BF16), (8, 2, 64, FP16), (8, 2, 96, BF16), (4, 1, 256, FP16), (16, 4, 128, FP16), (4, 1, 64, BF16),
          (12, 2, 64, BF16)]


def taken(step):
    """Whether the step's plan has prompts."""
    hits = [v for k, v in step.meta.get("_schedules", {}).items() if k[0] == "prompts4"]
    return len(hits) == 1 and hits[0] is not None


@pytest.mark.parametrize("hq,hkv,d,dtype", SHAPES)
@pytest.mark.parametrize("bs", [16, 48])
def test_prompts_beside_other_rows(cuda, sea, hq, hkv, d, dtype, bs):
    step = Step(sea, cuda, ROWS, hq, hkv, d, dtype, bs=bs)
    for causal in (True, False):
        announce("prompts", hq, hkv, d, dtype, bs, causal)
        o, l = step.call(sea, causal)
        assert taken(step)
        step.check(o, l, causal)
        o2, l2 = step.call(sea, causal)  # from the plan that is there
        step.check(o2, l2, causal)
    q = torch.randn(step.total, hq + 3, d + 1, device=cuda).to(dtype)[:, 1:hq + 1, :d]
    if dtype is not FP32 and d % 8 == 0:
        announce("prompts, strided queries", hq, hkv, d, dtype, bs)
        q = q.contiguous().transpose(0, 1).contiguous().transpose(0, 1)
    step.check(*step.call(sea, q=q), q=q)


@pytest.mark.parametrize("hq,hkv,d,dtype", SHAPES)
def test_nan_in_prompts(cuda, sea, hq, hkv, d, dtype):
    step = Step(sea, cuda, ROWS + [(140, 9000, 8860)], hq, hkv, d, dtype)
    bad = [(1, 260, 1, 3), (1, 399, 0, 40), (3, 64, 1, d - 1), (3, 100, 0, 0), (2, 75, 1, 5), (6, 0, 1, 33), (7, 8300, 1, 1),
           (7, 8990, 0, 2)]  # row, key, K or V, element
    bt = step.meta["block_table"].cpu().numpy()
    for r, key, kv, el in bad:
        slot = torch.tensor([int(bt[r, key // 16]) * 16 + key % 16], device=cuda)
        now = [x.clone() for x in step.cache.read(0, slot)]
        now[kv][0, :, el] = math.nan
        step.cache.write(now[0].unsqueeze(0).transpose(1, 2), now[1].unsqueeze(0).transpose(1, 2), 0, slot)
        step.keys[r][kv][key, :, el // 32 * 32:el // 32 * 32 + 32] = math.nan
    for causal in (True, False):
        announce("NaN in prompts", hq, hkv, d, dtype, causal)
        o, l = step.call(sea, causal)
        assert taken(step)
        want, _, _ = step.expected(causal)
        assert np.isnan(want).any() and not np.isnan(want).all()
        step.check(o, l, causal)


def test_streams_and_captures(cuda, sea):
    step = Step(sea, cuda, ROWS, 8, 2, 128, BF16)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    outs = []
    for s in streams * 2:
        with torch.cuda.stream(s):
            announce("prompts on a stream")
            outs.append(step.call(sea))
    torch.cuda.synchronize()
    for out in outs:
        step.check(*out)
    graphs = []
    for fresh in (False, True):  # planned before, and a step's first call
        if fresh:
            step.meta = {k: v for k, v in step.meta.items() if not k.startswith("_")}
        g = torch.cuda.CUDAGraph()
        announce("prompts captured", fresh)
        with torch.cuda.graph(g):
            out = step.call(sea)
        assert taken(step) != fresh
        graphs.append((g, out, step.meta))
    for _ in range(3):
        for g, out, _ in graphs:
            out[0].zero_()
            out[1].zero_()
            announce("replay")
            g.replay()
        step.check(*step.call(sea))
        torch.cuda.synchronize()
        for g, out, _ in graphs:
            step.check(*out)


def test_what_decides(cuda, sea, monkeypatch):
    kv4 = sea_module("kv_cache_4bit")
    for hq, dtype in ((8, FP32), (34, BF16)):  # (17 heads to a kv head)
        step = Step(sea, cuda, ROWS, hq, 2, 64, dtype)
        announce("no prompts", hq, dtype)
        step.check(*step.call(sea))
        assert not taken(step)
    step = Step(sea, cuda, ROWS, 8, 2, 64, BF16)
    step.meta["host_block_table"] = step.meta["host_block_table"][:, :3]  # shorter than the rows
    step.check(*step.call(sea))
    assert not taken(step)
    step = Step(sea, cuda, [(1, 300, 299), (20, 40, 20)], 8, 2, 64, BF16)
    step.check(*step.call(sea))
    assert not taken(step)
    step = Step(sea, cuda, [(kv4.PROMPT_PAIRS // 4, 300, 300 - kv4.PROMPT_PAIRS // 4)], 8, 2, 64, BF16)
    o, l = step.call(sea)
    assert taken(step)
    step.check(o, l)
    step.meta = {k: v for k, v in step.meta.items() if not k.startswith(("host_", "_"))}
    announce("prompts without host lengths")
    o2, l2 = step.call(sea)
    assert not taken(step)
    step.check(o2, l2)
    assert np.abs(f64(o) - f64(o2)).max() < 0.05
    monkeypatch.undo()
    for n in (False, True):  # operations of all prompts below and at the bound
        step = Step(sea, cuda, [(64, 1024 + 128, 1024 + 64)] * 8, 64, 8, 128, BF16)
        monkeypatch.setattr(kv4, "PROMPT_FLOPS", 8 * 4 * 64 * 128 * 64 * 1120 * (2 if not n else 1))
        announce("prompts' operations", n)
        step.check(*step.call(sea))
        assert taken(step) == n
        native = sea_module("_lib").native().attention4(step.q, step.cache.blocks(0), step.meta, 64, 8, step.scale, True,
                                                         sea_module("paged_attention_kernel")._WORKSPACES, kv4.PROMPT_PAIRS)
        assert (native is not None) == (not n)
