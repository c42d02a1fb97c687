"""Attention of drafted trees over the latent cache on a B200, against the
formula in 64 bits (tests/tree_ref.py)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.tree_ref import Case, check

pytestmark = pytest.mark.gpu


# lengths around the 64-row tiles, empty caches, node counts around the groups of four
SHAPES = [
    ([0], [1]), ([1], [1]), ([0], [5]), ([63], [1]), ([64], [1]), ([65], [2]), ([60], [4]), ([61], [4]),
    ([127], [64]), ([128], [64]), ([0], [64]), ([1000], [3]), ([1024], [8]), ([4099], [17]),
    ([0, 1, 64, 700], [1, 2, 3, 4]), ([513, 0, 77, 2050, 5], [13, 1, 64, 4, 7]), ([300] * 20, [8] * 20),
    ([9, 40, 3000], [0, 6, 0]), ([20000], [4]), ([33000, 100], [9, 33]),
]


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("lens,nodes", SHAPES)
def test_against_64_bits(K, torch_cuda, lens, nodes, q8):
    c = Case(lens, nodes, q8=q8, seed=len(lens) * 1000 + lens[0] + sum(nodes))
    plan = c.plan(K)
    c.run(plan)
    assert plan.check() == 0
    check(c)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("nh,R,DR", [(2, 6, 2), (5, 40, 8), (16, 512, 32), (1, 1, 2), (16, 256, 64)])
def test_other_shapes(K, torch_cuda, nh, R, DR, q8):
    c = Case([70, 0, 1500], [5, 9, 2], q8=q8, nh=nh, R=R, DR=DR, seed=R)
    plan = c.plan(K)
    c.run(plan)
    assert plan.check() == 0
    check(c)


@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("shape", [(16, 512, 64), (3, 24, 8)])
def test_masks_that_leave_nodes_empty(K, torch_cuda, shape, q8):
    nh, R, DR = shape
    c = Case([0, 0, 50, 200], [6, 64, 11, 4], q8=q8, nh=nh, R=R, DR=DR, seed=5, hide=0.4)
    plan = c.plan(K)
    c.run(plan)
    assert plan.check() == 0
    check(c)


@pytest.mark.parametrize("shape", [(16, 512, 64), (3, 24, 8)])
def test_bits_behind_the_last_node_are_ignored(K, torch_cuda, shape):
    nh, R, DR = shape
    c = Case([100, 30], [5, 64], nh=nh, R=R, DR=DR, seed=6)
    plan = c.plan(K)
    c.run(plan)
    want = c.out.clone(), c.lse.clone()
    c.mask[:5] |= -(1 << 5)
    c.run(plan)
    assert torch.equal(c.out, want[0]) and torch.equal(c.lse, want[1])


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("q8", [False, True])
@pytest.mark.parametrize("shape", [(16, 512, 64), (3, 24, 8)])
def test_hidden_rows_may_hold_anything(K, torch_cuda, shape, q8, value):
    """Rows between the sequences, and drafted rows that a node does not see."""
    nh, R, DR = shape
    c = Case([70, 64, 5], [9, 7, 64], q8=q8, nh=nh, R=R, DR=DR, seed=8)
    bad = [70 + 6, 64 + 2, 5 + 33]  # in rows of their sequences
    skip = set()
    first = 0
    for b, t in enumerate(c.nodes):
        for i in range(t):
            if bad[b] in c.seen(b, i):
                skip.add(first + i)
        first += t
    used = torch.zeros(c.rows, dtype=torch.bool)
    for a, n, t in zip(c.row0, c.lens, c.nodes):
        used[a:a + n + t] = True
    at = torch.tensor([c.row0[b] + bad[b] for b in range(3)] + (~used).nonzero().flatten().tolist(), device="cuda")
    if q8:
        c.rope[at] = value
        c.lscale[at] = value
    else:
        c.kv[at] = value
    plan = c.plan(K)
    c.run(plan)
    assert plan.check() == 0
    clean = Case([70, 64, 5], [9, 7, 64], q8=q8, nh=nh, R=R, DR=DR, seed=8)
    clean.out, clean.lse = c.out, c.lse
    check(clean, skip)
    assert len(skip) < c.total
    if value != value:  # a node that does see a row of NaN says so
        for node in skip:
            assert torch.isnan(c.out[node].float()).all() and torch.isnan(c.lse[node]).all()


def test_queries_that_are_not_finite_stay_by_themselves(K, torch_cuda):
    c = Case([130], [6], seed=9)
    c.q[2] = float("nan")
    c.q[3, 4, 100] = float("inf")
    plan = c.plan(K)
    c.run(plan)
    assert torch.isnan(c.out[2].float()).all() and torch.isnan(c.out[3, 4].float()).all()
    kept = c.out.clone(), c.lse.clone()
    c.q[2:4] = 0
    c.run(plan)
    check(c)
    keep = [0, 1, 4, 5]
    assert torch.equal(c.out[keep], kept[0][keep]) and torch.equal(c.lse[keep], kept[1][keep])


@pytest.mark.parametrize("q8", [False, True])
def test_sharp_and_flat_scores(K, torch_cuda, q8):
    """Scores of +-hundreds (one row takes all the weight, the maximum keeps moving) and a scale of 0."""
    c = Case([2000, 300], [6, 3], q8=q8, seed=10, sd=20.0)
    plan = c.plan(K)
    c.run(plan)
    check(c)
    c.run(plan, scale=0.0)
    check(c, scale=0.0)


@pytest.mark.parametrize("q8", [False, True])
def test_same_answer_every_time_and_whatever_runs_beside(K, torch_cuda, q8):
    c = Case([5000, 0, 129], [11, 3, 64], q8=q8, seed=11)
    d = Case([700], [9], q8=q8, seed=12)
    pc, pd = c.plan(K), d.plan(K)
    c.run(pc)
    d.run(pd)
    torch.cuda.synchronize()
    want = [t.clone() for t in (c.out, c.lse, d.out, d.lse)]
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(10):
        for t in (c.out, c.lse, d.out, d.lse):
            t.fill_(3)
        torch.cuda.synchronize()
        c.run(pc, stream=s1.cuda_stream)
        d.run(pd, stream=s2.cuda_stream)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, (c.out, c.lse, d.out, d.lse)))
    assert pc.check() == 0 and pd.check() == 0


@pytest.mark.parametrize("q8", [False, True])
def test_captured_and_replayed_with_new_inputs(K, torch_cuda, q8):
    c = Case([3000, 40], [5, 30], q8=q8, seed=13)
    plan = c.plan(K)
    c.run(plan)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        c.run(plan, stream=torch.cuda.current_stream().cuda_stream)
    for seed in (21, 22):
        new = Case([3000, 40], [5, 30], q8=q8, seed=seed)
        c.q.copy_(new.q)
        c.mask.copy_(new.mask)
        c.words = new.words
        c.out.fill_(3)
        graph.replay()
        torch.cuda.synchronize()
        check(c)


def test_without_lse_and_with_few_ctas(K, torch_cuda):
    c = Case([900, 10], [7, 2], seed=14)
    plan = c.plan(K)
    c.run(plan)
    lse = c.lse.clone()
    c.lse.fill_(5)
    c.run(plan, lse=False)
    assert torch.all(c.lse == 5)
    c.lse.copy_(lse)
    check(c)
    for n in (1, 3):
        few = c.plan(K, max_ctas=n)
        assert few.info()["ctas"] <= n
        c.run(few)
        check(c)


def test_only_the_outputs_are_written(K, torch_cuda):
    c = Case([77, 500], [5, 6], seed=15)
    big = torch.full((c.total + 2, 16, 512), 9.0, device="cuda", dtype=torch.bfloat16)
    lse = torch.full((c.total + 2, 16), 9.0, device="cuda")
    c.out, c.lse = big[1:-1], lse[1:-1]
    kv = c.kv.clone()
    c.run(c.plan(K))
    check(c)
    assert torch.equal(kv, c.kv)
    assert torch.all(big[0] == 9) and torch.all(big[-1] == 9) and torch.all(lse[0] == 9) and torch.all(lse[-1] == 9)


def test_refusals(K, torch_cuda):
    c = Case([70], [3], seed=16)
    plan = c.plan(K)
    good = dict(out=c.out, lse=c.lse, q=c.q, mask=c.mask, kv=c.kv, rows=c.rows)
    plan.attend_bf16(**good)
    for key in ("out", "q", "mask", "kv"):
        with pytest.raises(K.KvlError):
            plan.attend_bf16(**{**good, key: None})
    with pytest.raises(K.KvlError, match="pool row"):
        plan.attend_bf16(**{**good, "rows": c.row0[0] + 72})
    with pytest.raises(K.KvlError):
        plan.attend_bf16(**{**good, "rope_dim": 63})
    with pytest.raises(K.KvlError):
        plan.attend_q8(c.out, c.lse, c.q, c.mask, None, None, None, c.rows)
    odd = torch.zeros(c.kv.numel() + 8, device="cuda", dtype=torch.bfloat16)
    for key in ("q", "kv", "out"):
        with pytest.raises(K.KvlError, match="align"):
            plan.attend_bf16(**{**good, key: odd[1:]})
    with pytest.raises(K.KvlError, match="align"):
        plan.attend_bf16(**{**good, "mask": c.q.view(torch.int32).flatten()[1:]})
    plan.attend_bf16(**good)
    assert plan.check() == 0
    check(c)
