"""Rows of latent pools that are accepted, forked and compacted, bit for bit."""
from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def bf16_pools(n, rows, width=576, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randint(-32768, 32768, (n, rows, width), device="cuda", dtype=torch.int16, generator=g)


def q8_pools(n, rows, R=512, DR=64, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    lat = torch.randint(-128, 128, (n, rows, R), device="cuda", dtype=torch.int8, generator=g)
    sc = torch.randint(-2 ** 31, 2 ** 31 - 1, (n, rows), device="cuda", dtype=torch.int32, generator=g)
    rope = torch.randint(-32768, 32768, (n, rows, DR), device="cuda", dtype=torch.int16, generator=g)
    return [lat, sc, rope]


def pools(K, kind, n, rows, R=512, DR=64, seed=0):
    """(the arrays, the pool set)"""
    if kind == "bf16":
        kv = bf16_pools(n, rows, R + DR, seed)
        return [kv], K.PoolSet.bf16(kv, R, DR)
    a = q8_pools(n, rows, R, DR, seed)
    return a, K.PoolSet.q8(*a)


def moved(arrays, src, dst):
    want = [t.clone() for t in arrays]
    for w, t in zip(want, arrays):
        w[:, dst] = t[:, src]
    return want


def same(arrays, want):
    return all(torch.equal(a, b) for a, b in zip(arrays, want))


@pytest.mark.parametrize("kind", ["bf16", "q8"])
@pytest.mark.parametrize("n,batch,nodes,R,DR", [(1, 1, 1, 512, 64), (1, 1, 8, 512, 64), (3, 5, 64, 512, 64),
                                                (64, 2, 13, 512, 64), (2, 70, 32, 512, 64), (2, 4, 20, 7, 2),
                                                (1, 3, 64, 36, 6)])
def test_accept(K, torch_cuda, kind, n, batch, nodes, R, DR):
    r = np.random.RandomState(nodes + batch)
    stride = 100
    a, ps = pools(K, kind, n, batch * stride, R, DR, seed=batch)
    path = r.randint(0, 64, (batch, nodes)).astype(np.int32)
    count = r.randint(0, nodes + 1, batch).astype(np.int32)
    count[-1] = nodes
    base = np.array([b * stride + r.randint(0, stride - 64) for b in range(batch)], np.int64)
    src, dst = [], []
    for b in range(batch):
        keep = np.sort(r.choice(64 if count[b] < nodes else nodes, count[b], replace=False))
        path[b, :count[b]] = keep
        src += list(base[b] + keep)
        dst += list(base[b] + np.arange(count[b]))
    want = moved(a, torch.tensor(src, device="cuda"), torch.tensor(dst, device="cuda"))
    kept = torch.full((batch,), 99, device="cuda", dtype=torch.int32)
    dev = [torch.from_numpy(x).cuda() for x in (base, path, count)]
    ps.tree_accept(*dev, kept)
    torch.cuda.synchronize()
    assert torch.equal(kept.cpu(), torch.from_numpy(count))
    assert same(a, want)


@pytest.mark.parametrize("kind", ["bf16", "q8"])
def test_accept_refuses_sequence_by_sequence(K, torch_cuda, kind):
    a, ps = pools(K, kind, 2, 400)
    path = torch.tensor([[1, 3, 5], [2, 2, 4], [4, 3, 5], [-1, 0, 1], [0, 1, 2], [0, 5, 90], [0, 5, 9], [3, 8, 9],
                         [0, 1, 2 ** 31 - 1]], dtype=torch.int32, device="cuda")
    base = torch.tensor([0, 20, 40, 60, 80, 350, 200, 205, 300], device="cuda")
    count = torch.tensor([3, 3, 3, 3, 3, 3, 3, 3, 3], dtype=torch.int32, device="cuda")
    kept = torch.zeros(9, dtype=torch.int32, device="cuda")
    want = moved(a, torch.tensor([1, 3, 5], device="cuda"), torch.tensor([0, 1, 2], device="cuda"))
    ps.tree_accept(base, path, count, kept)
    # 5, 8: past the pool; 6 and 7 share rows 205..209
    assert kept.tolist() == [3, -1, -1, -1, 3, -1, -1, -1, -1]
    assert same(a, want)
    count = torch.tensor([0, -1, 4, 3, 1, 1, 2, 1, 0], dtype=torch.int32, device="cuda")
    base = torch.tensor([0, 20, 40, -5, 399, 400, 50, 51, 2 ** 40], device="cuda")
    path[3] = torch.tensor([1, 2, 3], dtype=torch.int32)
    want = [t.clone() for t in a]
    ps.tree_accept(base, path, count, kept)
    assert kept.tolist() == [0, -1, -1, -1, 1, -1, -1, -1, 0]
    assert same(a, want)
    # the same sequence twice: nobody moves it
    ps.tree_accept(torch.tensor([10, 10], device="cuda"), torch.tensor([[1], [2]], dtype=torch.int32, device="cuda"),
                   torch.tensor([1, 1], dtype=torch.int32, device="cuda"), kept)
    assert kept[:2].tolist() == [-1, -1] and same(a, want)


def runs_to_rows(src, dst, count):
    s = [x for a, n in zip(src, count) for x in range(a, a + n)]
    d = [x for a, n in zip(dst, count) for x in range(a, a + n)]
    return torch.tensor(s, dtype=torch.long, device="cuda"), torch.tensor(d, dtype=torch.long, device="cuda")


MOVES = [
    ("one row", [5], [0], [1]),
    ("nothing", [5, 9], [5, 20], [7, 0]),
    ("fork", [0, 0, 0], [1000, 2100, 3300], [1000, 900, 1]),
    ("swap apart", [0, 500], [1000, 2000], [400, 77]),
    ("up, no overlap", [0], [3000], [1500]),
    ("slide by one", [1], [0], [3999]),
    ("slide by 33", [133], [100], [3500]),
    ("slide far", [1500], [0], [2500]),
    ("holes", [0, 100, 700, 705, 2000], [0, 90, 690, 695, 1000], [90, 600, 3, 200, 1900]),
    ("many short", list(range(1, 3001, 3)), list(range(0, 1000)), [1] * 1000),
]


@pytest.mark.parametrize("kind", ["bf16", "q8"])
@pytest.mark.parametrize("name,src,dst,count", MOVES, ids=[m[0] for m in MOVES])
@pytest.mark.parametrize("n,R,DR", [(1, 512, 64), (3, 512, 64), (2, 7, 2)])
def test_move(K, torch_cuda, kind, name, src, dst, count, n, R, DR):
    a, ps = pools(K, kind, n, 4600, R, DR, seed=n)
    plan = K.PoolMovePlan(src, dst, count)
    s, d = runs_to_rows(src, dst, count)
    for _ in range(3):  # the plan serves again, on the rows as they are by then
        want = moved(a, s, d)
        plan.move(ps)
        assert plan.check() == 0
        assert same(a, want)
    assert plan.info()["moved_rows"] == sum(c for x, y, c in zip(src, dst, count) if x != y)


@pytest.mark.parametrize("kind", ["bf16", "q8"])
def test_large_compaction_and_replay(K, torch_cuda, kind):
    """A pool far larger than what is in flight at once, moved by one row, then by a captured graph."""
    rows = 120000
    a, ps = pools(K, kind, 2, rows, seed=3)
    for shift in (1, 31, 5000):
        want = [torch.cat([t[:, shift:], t[:, rows - shift:]], 1) for t in a]
        plan = K.PoolMovePlan([shift], [0], [rows - shift])
        plan.move(ps)
        assert plan.check() == 0 and same(a, want)
    plan = K.PoolMovePlan([7], [3], [rows - 7])
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        plan.move(ps, stream=torch.cuda.current_stream().cuda_stream)
    for _ in range(3):
        want = [torch.cat([t[:, :3], t[:, 7:], t[:, rows - 4:]], 1) for t in a]
        graph.replay()
        torch.cuda.synchronize()
        assert plan.check() == 0 and same(a, want)


def test_pools_that_are_refused(K, torch_cuda):
    a = bf16_pools(2, 300)
    plan = K.PoolMovePlan([200], [0], [100])
    with pytest.raises(K.KvlError, match="overlap"):
        plan.move(K.PoolSet.bf16([a[0], a[0]]))
    with pytest.raises(K.KvlError, match="overlap"):
        plan.move(K.PoolSet.bf16([a.view(-1, 576)[:300], a.view(-1, 576)[299:599]]))
    with pytest.raises(K.KvlError, match="row 300"):
        plan.move(K.PoolSet.bf16([a[0][:299]]))
    with pytest.raises(K.KvlError, match="at once"):
        plan.move(K.PoolSet.bf16(bf16_pools(65, 300)))
    with pytest.raises(K.KvlError):
        plan.move(K.PoolSet.bf16([]))
    with pytest.raises(K.KvlError):
        K.PoolSet.bf16([a[0][:, :500]])
    before = a.clone()
    assert torch.equal(a, before)


@pytest.mark.parametrize("kind", ["bf16", "q8"])
@pytest.mark.parametrize("R,DR", [(1024, 64), (2000, 64), (512, 60), (16, 8), (3000, 8)])
@pytest.mark.parametrize("src,dst,count", [([3], [0], [700]), ([0, 50], [400, 600], [133, 90])])
def test_move_row_widths(K, torch_cuda, kind, R, DR, src, dst, count):
    """Rows that two, one or no ring of bulk copies holds, and rows that bulk copies cannot take."""
    a, ps = pools(K, kind, 2, 710, R, DR, seed=5)
    plan = K.PoolMovePlan(src, dst, count)
    want = moved(a, *runs_to_rows(src, dst, count))
    plan.move(ps)
    assert plan.check() == 0 and same(a, want)


@pytest.mark.parametrize("off", [1, 2, 4, 8])
def test_move_misaligned_pools(K, torch_cuda, off):
    flat = torch.randint(-32768, 32768, (300 * 576 + 8,), device="cuda", dtype=torch.int16)
    a = flat[off:off + 300 * 576].view(300, 576)
    before, rest = a.clone(), flat.clone()
    K.PoolMovePlan([37], [2], [260]).move(K.PoolSet.bf16([a]))
    assert torch.equal(a[2:262], before[37:297]) and torch.equal(a[:2], before[:2]) and torch.equal(a[262:], before[262:])
    assert torch.equal(flat[:off], rest[:off]) and torch.equal(flat[off + 300 * 576:], rest[off + 300 * 576:])


def test_rows_too_wide_for_a_tile(K, torch_cuda):
    a = torch.zeros(4, 4096, dtype=torch.int16, device="cuda")
    with pytest.raises(K.KvlError, match="rows of 8192 bytes"):
        K.PoolMovePlan([1], [0], [3]).move(K.PoolSet.bf16([a], 4032, 64))
