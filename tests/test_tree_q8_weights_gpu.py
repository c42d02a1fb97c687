"""The softmax weights of the Q8 tree attend have 16 bits: an output is off by the rounding of its own and little else.

Bound of an element, against the formula in 64 bits: a weight enters the product as two bf16 parts, the first off by
2^-8 of it at most and the second by 2^-8 of that, so by 2^-16 in all; the scores' error ds and the sums as in
tests.tree_ref.check, with twice as many terms; the output's own rounding 2^-8 of it.
"""
from __future__ import annotations

import pytest
import torch

from tests.tree_ref import HALF_BF16, HALF_F32, Case

pytestmark = pytest.mark.gpu


def check(c):
    first = 0
    for b, t in enumerate(c.nodes):
        lat, rope = c.rows64(b)
        for i in range(t):
            node, idx = first + i, c.seen(b, i)
            out = c.out[node].double()
            if not idx:
                assert torch.all(out == 0), (b, i)
                continue
            j = torch.tensor(idx, device=lat.device)
            kl, kr = lat[j], rope[j]
            q = c.q[node].double()
            ql, qr = q[:, :c.R], q[:, c.R:]
            s = (ql @ kl.T + qr @ kr.T) * c.scale
            p = torch.softmax(s, -1)
            want, mass = p @ kl, p @ kl.abs()
            size = (ql.abs() @ kl.abs().T + qr.abs() @ kr.abs().T).amax(-1) * c.scale
            ds = 2 * (c.R + c.DR + 1) * HALF_F32 * size + 2.0 ** -22
            tol = (2.0 ** -16 + 3 * ds[:, None] + 4 * len(idx) * HALF_F32) * mass * 1.02 + HALF_BF16 * want.abs() * 1.02
            bad = ((out - want).abs() / (tol + 1e-30)).max().item()
            assert bad <= 1.0, (b, i, bad)
        first += t


@pytest.mark.parametrize("lens,nodes,ctas", [
    ([3] * 31, [3] * 31, 0), ([17] * 10, [1, 1, 1, 2, 2, 1, 1, 1, 1, 2], 0), ([0], [64], 0), ([64], [4], 0),
    ([200, 0, 63], [9, 64, 1], 0), ([900], [8], 0), ([44] * 12, [4] * 12, 1), ([108] * 9, [4] * 9, 2), ([1500], [5], 1),
    ([20, 300, 70, 5], [4, 4, 4, 4], 1)])
@pytest.mark.parametrize("hide", [0.0, 0.3])
def test_weights_have_sixteen_bits(K, torch_cuda, lens, nodes, ctas, hide):
    c = Case(lens, nodes, q8=True, seed=sum(lens) + len(lens), hide=hide)
    plan = c.plan(K, max_ctas=ctas)
    for _ in range(3):
        c.out.fill_(3)
        c.run(plan)
        assert plan.check() == 0
    check(c)


def test_weights_of_other_shapes(K, torch_cuda):
    c = Case([70, 0], [5, 9], q8=True, nh=3, R=24, DR=8, seed=4)
    c.run(c.plan(K))
    check(c)
