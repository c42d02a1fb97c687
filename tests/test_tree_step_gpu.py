"""A layer's step for drafted trees, and a round of speculative decoding put
together from it, the acceptance of a path and the moves of rows, against the
single-token decode step on the same weights and rows.

Tolerance of an output (tests.parity): rel-L2 <= 1e-2, max-abs <= 2e-2.  On its
way it is rounded to bf16 six times (q_nope, the absorbed query, the softmax
weights, the mix, the V up-projection's output, and the activations), each off
by at most 2^-8 and by 2^-8 / sqrt(3) x 0.72 = 1.6e-3 in the root mean square;
the decode step it is held against does four of them.  Independent errors of
1.6e-3 add up to sqrt(10) x 1.6e-3 = 5.1e-3.
"""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest
import torch

from tests.parity import assert_close

pytestmark = pytest.mark.gpu

H, NH, R, DR = 2048, 16, 512, 64
GAP = 5  # rows of others between the sequences


class Model:
    def __init__(self, K, layers, seed):
        self.K, self.lib = K, K.load()
        self.cfg = K.make_config(H, NH, 128, DR, 128, R, 1e-5, 50000.0)
        self.keep, self.w = [], []
        for i in range(layers):
            w = K.random_weights(self.cfg, seed + i, 0.02, norm_std=0.05)
            ts = [torch.from_numpy(a.view(np.int16)).cuda() for a in w.arrays]
            self.keep.append(ts)
            self.w.append(K.KvlMlaDeviceWeights(*[t.data_ptr() for t in ts]))

    def workspace(self, n):
        return torch.empty(self.lib.kvl_mla_decode_step_workspace_bytes(C.byref(self.cfg), n), dtype=torch.uint8,
                           device="cuda")


class Pool:
    """The latent pools of all layers."""

    def __init__(self, layers, rows, q8, seed):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.q8, self.rows = q8, rows
        if q8:
            self.arrays = [torch.randint(-127, 128, (layers, rows, R), device="cuda", dtype=torch.int8, generator=g),
                           torch.rand(layers, rows, device="cuda", generator=g) * 0.019 + 0.001,
                           torch.randn(layers, rows, DR, device="cuda", generator=g).to(torch.bfloat16)]
        else:
            self.arrays = [torch.randn(layers, rows, R + DR, device="cuda", generator=g).to(torch.bfloat16)]

    def clone(self):
        p = object.__new__(Pool)
        p.q8, p.rows, p.arrays = self.q8, self.rows, [a.clone() for a in self.arrays]
        return p

    def values(self, layer, a, b):
        if self.q8:
            lat = self.arrays[0][layer, a:b].float() * self.arrays[1][layer, a:b, None]
            return torch.cat([lat, self.arrays[2][layer, a:b].float()], 1).cpu().numpy()
        return self.arrays[0][layer, a:b].float().cpu().numpy()

    def set(self, K):
        return K.PoolSet.q8(*self.arrays) if self.q8 else K.PoolSet.bf16(self.arrays[0])


def tree_step(m, pool, layer, plan, x, mask, pos, out=None, ws=None, stream=0, rows=None):
    out = torch.empty_like(x) if out is None else out
    ws = m.workspace(x.shape[0]) if ws is None else ws
    step = plan.step_q8 if pool.q8 else plan.step_bf16
    step(m.cfg, m.w[layer], out, x, mask, pos, *[a[layer] for a in pool.arrays], pool.rows if rows is None else rows, ws,
         stream=stream)
    return out


def decode(m, pool, layer, row0, lens, x):
    """One token for every sequence behind its `lens` rows."""
    plan = m.K.AttendPlan([n + 1 for n in lens], row0, NH, R)
    out, ws, B = torch.empty_like(x), m.workspace(len(lens)), len(lens)
    d_row = torch.tensor([a + n for a, n in zip(row0, lens)], dtype=torch.int64, device="cuda")
    d_pos = torch.tensor(lens, dtype=torch.int32, device="cuda")
    fn = m.lib.kvl_mla_decode_step_q8 if pool.q8 else m.lib.kvl_mla_decode_step_bf16
    rc = fn(C.byref(m.cfg), C.byref(m.w[layer]), plan.h, out.data_ptr(), x.data_ptr(),
            *[a[layer].data_ptr() for a in pool.arrays], pool.rows, d_row.data_ptr(), d_pos.data_ptr(), B, ws.data_ptr(),
            C.c_void_p(0))
    assert rc == 0, m.K.last_error()
    assert plan.check() == 0, m.K.last_error()
    return out


def assert_rows(p, layer, a, other, b, n):
    """The same rows, computed with sums in another order: an element that lies
    between two values of its type may have become either of them.  One step of
    bf16 is at most 2^-7 of the value, one of the row quantiser the row's largest
    value / 127 (whose own error, 1e-4 relative, makes 0.0127 of a step)."""
    x, y = p.values(layer, a, a + n), other.values(layer, b, b + n)
    step = 2.0 ** -7 * np.maximum(np.abs(x), np.abs(y)) + 1e-4
    if p.q8:
        step[:, :R] = 1.02 * np.abs(y[:, :R]).max(1, keepdims=True) / 127
    assert np.all(np.abs(x - y) <= step), (a, b, np.abs(x - y).max())


def layout(lens, room):
    row0, at = [], GAP
    for n, t in zip(lens, room):
        row0.append(at)
        at += n + t + GAP
    return row0, at + 64


def trees(K, nodes, seed):
    r = np.random.RandomState(seed)
    parents = [np.array([-1 if i == 0 else r.randint(-1, i) for i in range(t)], np.int32) for t in nodes]
    words = np.concatenate([K.tree_mask(p) for p in parents if len(p)])
    return parents, torch.from_numpy(words.view(np.int64)).cuda()


def path_to(parent, i):
    p = [i]
    while parent[p[0]] >= 0:
        p.insert(0, int(parent[p[0]]))
    return p


@pytest.mark.parametrize("q8", [False, True], ids=["bf16", "q8"])
@pytest.mark.parametrize("lens,nodes", [([100], [1]), ([0, 37, 260], [3, 0, 8]), ([5, 64, 63, 0, 700], [4, 5, 1, 7, 33]),
                                        ([90] * 40, [8] * 40), ([20] * 34, [64] * 34)])
def test_step_decodes_every_path(K, torch_cuda, q8, lens, nodes):
    m = Model(K, 1, 21)
    row0, rows = layout(lens, nodes)
    pool = Pool(1, rows, q8, 22)
    before = pool.clone()
    parents, mask = trees(K, nodes, 23)
    depth = [len(path_to(p, i)) - 1 for p in parents for i in range(len(p))]
    seq = [b for b, t in enumerate(nodes) for _ in range(t)]
    at = [i for t in nodes for i in range(t)]
    pos = torch.tensor([lens[b] + d for b, d in zip(seq, depth)], dtype=torch.int32, device="cuda")
    x = torch.randn(sum(nodes), H, device="cuda").to(torch.bfloat16).float()
    plan = K.TreePlan(lens, nodes, row0)
    out = tree_step(m, pool, 0, plan, x, mask, pos)
    assert plan.check() == 0, K.last_error()
    # a decode of every node on its own copy of the cache and its ancestors' rows
    have = [lens[b] + d for b, d in zip(seq, depth)]
    copy0, total = layout(have, [1] * len(have))
    copies = Pool(1, total, q8, 24)
    for k, (b, i) in enumerate(zip(seq, at)):
        src = list(range(row0[b], row0[b] + lens[b])) + [row0[b] + lens[b] + j for j in path_to(parents[b], i)[:-1]]
        for c, p in zip(copies.arrays, pool.arrays):
            c[0, copy0[k]:copy0[k] + len(src)] = p[0, src]
    # positions of the copies: cached length plus depth, the rows they have
    want = decode(m, copies, 0, copy0, have, x)
    for k, (b, i) in enumerate(zip(seq, at)):
        assert_close(out[k].cpu().numpy(), want[k].cpu().numpy(), what=f"node {i} of sequence {b}")
        r = row0[b] + lens[b] + i
        assert_rows(pool, 0, r, copies, copy0[k] + have[k], 1)
    drafted = torch.zeros(rows, dtype=torch.bool, device="cuda")
    for b in range(len(lens)):
        drafted[row0[b] + lens[b]:row0[b] + lens[b] + nodes[b]] = True
    for a, b in zip(pool.arrays, before.arrays):
        assert torch.equal(a[:, ~drafted], b[:, ~drafted])


@pytest.mark.parametrize("q8", [False, True], ids=["bf16", "q8"])
def test_round_of_speculation(K, torch_cuda, q8):
    """Draft, verify, accept, decode on; fork a sequence; drop one and compact."""
    layers, lens, nodes = 2, [3, 150, 64], [9, 6, 4]
    m = Model(K, layers, 31)
    row0, rows = layout(lens, [t + 4 for t in nodes])
    rows += 2 * 20
    pool = Pool(layers, rows, q8, 32)
    serial = pool.clone()
    parents, mask = trees(K, nodes, 33)
    first = np.concatenate([[0], np.cumsum(nodes)[:-1]])
    pos = torch.tensor([lens[b] + len(path_to(parents[b], i)) - 1 for b in range(3) for i in range(nodes[b])],
                       dtype=torch.int32, device="cuda")
    x = torch.randn(layers, sum(nodes), H, device="cuda").to(torch.bfloat16).float()
    plan = K.TreePlan(lens, nodes, row0)
    out = [tree_step(m, pool, i, plan, x[i], mask, pos) for i in range(layers)]
    assert plan.check() == 0, K.last_error()
    # accepted: the longest path, the root alone, nothing
    best = max((path_to(parents[0], i) for i in range(nodes[0])), key=len)
    paths = [best, [0], []]
    path = torch.zeros(3, max(nodes), dtype=torch.int32)
    for b, p in enumerate(paths):
        path[b, :len(p)] = torch.tensor(p, dtype=torch.int32)
    count = torch.tensor([len(p) for p in paths], dtype=torch.int32).cuda()
    kept = torch.empty(3, dtype=torch.int32, device="cuda")
    base = torch.tensor([a + n for a, n in zip(row0, lens)], dtype=torch.int64, device="cuda")
    pools = pool.set(K)
    pools.tree_accept(base, path.cuda(), count, kept)
    assert torch.equal(kept, count)
    # the accepted tokens one at a time
    now = list(lens)
    for j in range(max(map(len, paths))):
        for b, p in enumerate(paths):
            if j < len(p):
                for i in range(layers):
                    k = first[b] + p[j]
                    want = decode(m, serial, i, [row0[b]], [now[b]], x[i, k:k + 1].contiguous())
                    assert_close(out[i][k].cpu().numpy(), want[0].cpu().numpy(), what=f"token {j} of sequence {b}")
                now[b] += 1
    for b in range(3):
        for i in range(layers):
            assert_rows(pool, i, row0[b], serial, row0[b], now[b])
    # the next token of every sequence
    y = torch.randn(3, H, device="cuda").to(torch.bfloat16).float()
    after = [decode(m, pool.clone(), i, row0, now, y) for i in range(layers)]
    for i in range(layers):
        assert_close(after[i].cpu().numpy(), decode(m, serial, i, row0, now, y).cpu().numpy(), what="next token")
    # two forks of sequence 0 at the pool's end answer as it does
    forks = [rows - 40, rows - 20]
    assert now[0] + 1 < 20
    move = K.PoolMovePlan([row0[0]] * 2, forks, [now[0]] * 2)
    assert not move.info()["compaction"]
    move.move(pools)
    for i in range(layers):
        got = decode(m, pool.clone(), i, [row0[0]] + forks, [now[0]] * 3, y[:1].expand(3, H).contiguous())
        assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])
    # sequence 1 ends: the others slide together, one free row behind each
    order = [row0[0], row0[2]] + forks
    size = [now[0], now[2], now[0], now[0]]
    to, at = [], row0[0]
    for n in size:
        to.append(at)
        at += n + 1
    token = torch.stack([y[0], y[2], y[0], y[0]])
    was = [decode(m, pool.clone(), i, order, size, token) for i in range(layers)]
    move = K.PoolMovePlan(order, to, size)
    move.move(pools)
    assert move.check() == 0, K.last_error()
    for i in range(layers):
        assert torch.equal(decode(m, pool.clone(), i, to, size, token), was[i])


@pytest.mark.parametrize("q8", [False, True], ids=["bf16", "q8"])
def test_captured_round(K, torch_cuda, q8):
    lens, nodes, layers = [40, 7], [8, 5], 2
    m = Model(K, layers, 41)
    row0, rows = layout(lens, nodes)
    pool = Pool(layers, rows, q8, 42)
    start = pool.clone()
    parents, mask = trees(K, nodes, 43)
    pos = torch.tensor([lens[b] + len(path_to(parents[b], i)) - 1 for b in range(2) for i in range(nodes[b])],
                       dtype=torch.int32, device="cuda")
    x = torch.randn(layers, sum(nodes), H, device="cuda")
    plan = K.TreePlan(lens, nodes, row0)
    paths = [path_to(parents[0], 7), path_to(parents[1], 4)]
    path = torch.tensor([(p + [0] * 8)[:8] for p in paths], dtype=torch.int32).cuda()
    count = torch.tensor([len(p) for p in paths], dtype=torch.int32).cuda()
    base = torch.tensor([a + n for a, n in zip(row0, lens)], dtype=torch.int64, device="cuda")
    kept = torch.empty(2, dtype=torch.int32, device="cuda")
    out = torch.empty(layers, sum(nodes), H, device="cuda")
    ws, pools = m.workspace(sum(nodes)), pool.set(K)

    def a_round(stream):
        for i in range(layers):
            tree_step(m, pool, i, plan, x[i], mask, pos, out=out[i], ws=ws, stream=stream)
        pools.tree_accept(base, path, count, kept, stream=stream)

    a_round(torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    eager, after = out.clone(), pool.clone()
    assert torch.equal(kept, count)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a_round(torch.cuda.current_stream().cuda_stream)
    for _ in range(2):
        for a, b in zip(pool.arrays, start.arrays):
            a.copy_(b)
        out.zero_()
        kept.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert plan.check() == 0, K.last_error()
        assert torch.equal(out, eager) and torch.equal(kept, count)
        for a, b in zip(pool.arrays, after.arrays):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    del graph


def test_step_refusals(K, torch_cuda):
    lens, nodes = [40], [4]
    m = Model(K, 1, 51)
    row0, rows = layout(lens, nodes)
    pool = Pool(1, rows, False, 52)
    before = pool.clone()
    parents, mask = trees(K, nodes, 53)
    pos = torch.zeros(4, dtype=torch.int32, device="cuda")
    x = torch.zeros(4, H, device="cuda")
    plan = K.TreePlan(lens, nodes, row0)
    wide = torch.empty(4 * H + 1, device="cuda")
    with pytest.raises(K.KvlError, match="ends at pool row"):
        tree_step(m, pool, 0, plan, x, mask, pos, rows=row0[0] + 43)
    with pytest.raises(K.KvlError, match="aligned"):
        tree_step(m, pool, 0, plan, x, mask, pos, out=wide[1:])
    with pytest.raises(K.KvlError, match="aligned"):
        tree_step(m, pool, 0, plan, x, mask, pos, ws=m.workspace(5)[4:])
    with pytest.raises(K.KvlError, match="the plan is for 8 heads"):
        tree_step(m, pool, 0, K.TreePlan(lens, nodes, row0, num_heads=8), x, mask, pos)
    twice = K.TreePlan([40, 38], [2, 4], [row0[0], row0[0]])
    with pytest.raises(K.KvlError, match="the same drafted row"):
        tree_step(m, pool, 0, twice, torch.zeros(6, H, device="cuda"), mask, pos)
    with pytest.raises(K.KvlError, match="arguments"):
        tree_step(m, pool, 0, plan, x, None, pos)
    torch.cuda.synchronize()
    assert torch.equal(pool.arrays[0], before.arrays[0])
