"""Drafted rows that hold an infinity or a NaN in single elements: a node that sees such a row gets what the formula
says, element by element, whatever the other nodes see (a head whose scores are all -inf: 0 and -inf); a node that does
not see it gets what it gets without it."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from tests.tree_ref import HALF_BF16, HALF_F32, Case

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


def formula(c, b, i, scale):
    """out, lse and the bound on out's error (tests.tree_ref.check) of one node in 64 bits; not finite where it says so."""
    lat, rope = c.rows64(b)
    j = torch.tensor(c.seen(b, i), device=lat.device)
    kl, kr = lat[j], rope[j]
    q = c.q[sum(c.nodes[:b]) + i].double()
    ql, qr = q[:, :c.R], q[:, c.R:]
    prod = torch.cat([ql[:, None] * kl[None], qr[:, None] * kr[None]], -1)  # no product is left out: 0 * inf is NaN
    s = prod.sum(-1) * scale
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse[:, None])
    want = torch.where(torch.isneginf(lse)[:, None], 0.0, (p[..., None] * kl[None]).sum(1))
    clean = torch.where(torch.isfinite(prod), prod.abs(), 0.0)
    size = clean.sum(-1).amax(-1) * abs(scale)
    ds = 2 * (c.R + c.DR + 1) * HALF_F32 * size + 2.0 ** -22
    mass = torch.nan_to_num(p) @ torch.where(torch.isfinite(kl), kl.abs(), 0.0)
    tol = (HALF_BF16 + 3 * ds[:, None] + 2 * len(j) * HALF_F32) * mass * 1.02 + HALF_BF16 * want.abs() * 1.02 + 1e-30
    return want, lse, tol


def check(c, scale):
    """The number of outputs that are not finite."""
    first = total = 0
    for b, t in enumerate(c.nodes):
        for i in range(t):
            if not c.seen(b, i):
                continue
            want, lse, tol = formula(c, b, i, scale)
            out, got = c.out[first + i].double(), c.lse[first + i].double()
            nan = ~torch.isfinite(want)
            assert torch.equal(nan, ~torch.isfinite(out)), (b, i)
            assert torch.all((out - want).abs()[~nan] <= tol[~nan]), (b, i)
            fin = torch.isfinite(lse)
            assert torch.equal(fin, torch.isfinite(got)), (b, i)
            assert torch.all((got - lse)[fin].abs() <= 1e-3), (b, i)
            total += int(nan.sum())
        first += t
    return total


# cached rows, nodes, the drafted row that is spoilt: in the tile of the last cached rows, in the next one, in a tile of
# its own, the first and the last of a tree
BATCHES = [([70], [9], [6]), ([60], [12], [5]), ([64], [7], [2]), ([0], [64], [33]), ([40, 3, 700], [4, 64, 7], [0, 63, 4]),
           ([5000], [6], [1])]


@pytest.mark.parametrize("value,at", [(INF, 7), (-INF, 300), (NAN, 511), (INF, 512), (INF, 575)])
@pytest.mark.parametrize("lens,nodes,bad", BATCHES)
@pytest.mark.parametrize("shape", [(16, 512, 64), (3, 24, 8)])
def test_one_element(K, torch_cuda, shape, lens, nodes, bad, value, at):
    nh, R, DR = shape
    at = at if nh == 16 else at % (R + DR)
    total = 0
    for scale, ctas in ((0.07, 0), (-0.07, 1)):
        c = Case(lens, nodes, nh=nh, R=R, DR=DR, seed=sum(lens) + at)
        plan = c.plan(K, max_ctas=ctas)
        c.run(plan, scale=scale)
        clean = c.out.clone(), c.lse.clone()
        c.q[:, ::3, at] = c.q[:, ::3, at].abs() + 0.1  # both signs of an infinite score among the heads
        c.q[:, 1::3, at] = -c.q[:, 1::3, at].abs() - 0.1
        # some nodes of a group see the row, others do not; then all see it
        for every in (False, True):
            first = 0
            for b, t in enumerate(nodes):
                for i in range(t):
                    w = int(c.words[first + i]) & ~(1 << bad[b])
                    c.words[first + i] = w | (1 << bad[b] if every or i % 2 == 0 else 0)
                c.kv[c.row0[b] + lens[b] + bad[b], at] = value
                first += t
            c.mask.copy_(torch.from_numpy(c.words.view(np.int64)))
            c.out.fill_(3)
            c.run(plan, scale=scale)
            assert plan.check() == 0
            total += check(c, scale)
    assert total > 0


def test_a_seeing_node_does_not_depend_on_the_others(K, torch_cuda):
    """Bit for bit, NaN for NaN: the node that sees the row, whatever the other three of its group see."""
    c = Case([100], [4], seed=3)
    plan = c.plan(K)
    c.kv[c.row0[0] + 102, 9] = INF
    c.q[1, :, 9] = -1.0  # all its scores of the row are -inf: weight 0, and 0 * inf in one element
    got = []
    for others in (0, 1 << 2):
        words = [1 | others, 2 | 1 << 2, 1 | others, 8 | others]
        c.words[:] = words
        c.mask.copy_(torch.from_numpy(c.words.view(np.int64)))
        c.q[[0, 2, 3], :, 9] = -1.0
        c.run(plan)
        assert plan.check() == 0
        got.append((c.out[1].clone(), c.lse[1].clone()))
    nan = torch.isnan(got[0][0].float())
    assert nan[:, 9].all() and nan.sum() == 16
    assert torch.equal(nan, torch.isnan(got[1][0].float())) and torch.equal(got[0][0][~nan], got[1][0][~nan])
    assert torch.equal(got[0][1], got[1][1])
