"""build_block_tables against token-by-token Python."""
import numpy as np
import pytest
import torch

import layer_ref as ref

pytestmark = pytest.mark.gpu


def case(cuda, sea, prior, q_lens, width, free, total, bs=16, seed=0, max_q=None):
    rng = np.random.default_rng(seed)
    r = len(prior)
    table = rng.integers(0, 1 << 20, (r, width)).astype(np.int32)
    free = np.asarray(free, dtype=np.int32)
    i32 = lambda x: torch.tensor(np.asarray(x), dtype=torch.int32, device=cuda)  # noqa: E731
    bt = i32(table)
    print("case: tables", r, width, len(free), total, bs, flush=True)
    want = ref.block_tables(table.tolist(), prior, q_lens, free.tolist(), total, bs)
    for _ in range(2):  # a second call finds the table filled
        meta = sea.build_block_tables(bt, i32(prior), i32(q_lens), i32(free), total,
                                      max(max(q_lens, default=0), 0) if max_q is None else max_q, block_size=bs)
        got = (bt, meta["k_lens"], meta["q_starts"], meta["slot_mapping"], meta["positions"], meta["blocks_taken"])
        for name, g, w in zip(("table", "k_lens", "q_starts", "slots", "positions", "taken"), got, want):
            assert np.array_equal(g.cpu().numpy().reshape(np.shape(w)), np.array(w)), name
    assert meta["block_table"] is bt and meta["total_query"] == total
    return meta


@pytest.mark.parametrize("rows", [1, 2, 63, 64, 65, 200, 1500])
@pytest.mark.parametrize("bs", [16, 1, 48])
def test_random_steps(cuda, sea, rows, bs):
    rng = np.random.default_rng(rows + bs)
    prior = rng.integers(0, 200, rows)
    q = np.where(rng.random(rows) < 0.7, 1, rng.integers(0, 90, rows))
    prior[rng.random(rows) < 0.2] //= bs
    width = int((prior + q).max() + bs - 1) // bs + 1
    need = int(((prior + q + bs - 1) // bs - (prior + bs - 1) // bs).sum())
    total = int(q.sum())
    case(cuda, sea, prior.tolist(), q.tolist(), width, rng.permutation(need + 7), total + (rows % 3) * 50, bs)


def test_edges(cuda, sea):
    case(cuda, sea, [0], [0], 1, [], 0)
    case(cuda, sea, [0, 5, 0], [0, 0, 0], 2, [3], 4)                          # no tokens at all
    case(cuda, sea, [0, 16, 15, 17], [16, 16, 1, 15], 3, range(10, 30), 48)   # ends on block borders
    case(cuda, sea, [0], [5000], 400, range(400), 5000)                       # one long prompt
    case(cuda, sea, [3, 40], [5000, 1], 400, range(400), 5001, max_q=1)       # max_q_len sizes the grid only
    case(cuda, sea, [-3, 4], [2, -7], 2, range(4), 2)                         # negative lengths count as 0
    case(cuda, sea, [10, 10, 10], [40, 40, 40], 4, [5, 6, 7, 8], 120)         # fewer free blocks than it takes
    case(cuda, sea, [10, 10], [40, 60], 3, range(9), 100)                     # a table too narrow
    case(cuda, sea, [10, 10], [40, 60], 5, range(9), 70)                      # fewer slots than tokens


def test_no_rows_and_refusals(cuda, sea):
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=cuda)  # noqa: E731
    meta = sea.build_block_tables(i32(0, 3), i32(0), i32(0), i32(2), 3, 0)
    assert meta["slot_mapping"].tolist() == [-1] * 3 and meta["positions"].tolist() == [0] * 3
    assert meta["blocks_taken"].tolist() == [0]
    good = (i32(2, 3), i32(2), i32(2), i32(4), 2, 1)
    for i, bad in ((0, i32(2)), (0, i32(2, 3).long()), (0, i32(3, 2).t()), (1, i32(3)), (2, i32(2, 1)), (2, i32(2).cpu()),
                   (3, i32(4).long()), (4, -1), (5, -1)):
        args = list(good)
        args[i] = bad
        with pytest.raises((ValueError, TypeError)):
            sea.build_block_tables(*args)


def test_streams_and_captures(cuda, sea):
    """A step's tables recorded once and replayed on lengths that change."""
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    prior, q, free, bt = i32([5, 31, 0]), i32([1, 1, 1]), i32(list(range(9, 40))), torch.zeros(3, 6, dtype=torch.int32, device=cuda)
    start = bt.clone()
    sea.build_block_tables(bt, prior, q, free, 20, 5)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        meta = sea.build_block_tables(bt, prior, q, free, 20, 5)
    for p, n in (([5, 31, 0], [1, 1, 1]), ([6, 32, 1], [5, 3, 0]), ([16, 2, 1], [2, 5, 5])):
        prior.copy_(i32(p))
        q.copy_(i32(n))
        bt.copy_(start)
        g.replay()
        torch.cuda.synchronize()
        want = ref.block_tables(start.tolist(), p, n, free.tolist(), 20, 16)
        assert bt.tolist() == want[0] and meta["slot_mapping"].tolist() == want[3]
        assert meta["positions"].tolist() == want[4] and meta["blocks_taken"].tolist() == [want[5]]
