"""A step for drafted trees writes no row that another sequence of its plan owns: sequences may share cached rows, and
a plan that drafts into another's rows is refused before anything is written."""
from __future__ import annotations

import pytest
import torch

from tests.test_tree_step_gpu import H, Model, Pool, tree_step, trees

pytestmark = pytest.mark.gpu

# (cached rows, drafted nodes, first rows) of a batch
REFUSED = [
    ([100, 50], [0, 8], [0, 0]),          # behind 50 rows of a prefix of 100: the other's rows 50..57
    ([100, 50], [4, 8], [0, 0]),
    ([50, 100], [8, 0], [0, 0]),          # the same, the other way round
    ([100, 20], [0, 8], [0, 73]),         # drafted rows 93..100: the first seven are the other's last
    ([20, 100], [8, 0], [0, 27]),         # one row of the other's
    ([20, 1], [8, 0], [0, 24]),           # a cache of one row within the drafted ones
    ([300, 10, 40], [0, 1, 3], [0, 400, 200]),  # a range that began long before
]
ALLOWED = [
    ([100, 100], [0, 8], [0, 0]),         # the whole cache shared, one of them drafts
    ([50, 20], [0, 8], [28, 0]),          # drafted rows that end where the other's cache begins
    ([50, 0, 20], [3, 0, 8], [100, 25, 0]),  # an empty cache has no rows
]


@pytest.mark.parametrize("q8", [False, True], ids=["bf16", "q8"])
@pytest.mark.parametrize("lens,nodes,row0", REFUSED + ALLOWED)
def test_drafted_rows_in_another_sequences_cache(K, torch_cuda, lens, nodes, row0, q8):
    m = Model(K, 1, 61)
    pool = Pool(1, 512, q8, 62)
    before = pool.clone()
    parents, mask = trees(K, nodes, 63)
    pos = torch.tensor([n for n, t in zip(lens, nodes) for _ in range(t)], dtype=torch.int32, device="cuda")
    x = torch.randn(sum(nodes), H, device="cuda")
    plan = K.TreePlan(lens, nodes, row0)
    keep = torch.ones(512, dtype=torch.bool, device="cuda")
    if (lens, nodes, row0) in REFUSED:
        with pytest.raises(K.KvlError, match="cached row of another"):
            tree_step(m, pool, 0, plan, x, mask, pos)
    else:
        tree_step(m, pool, 0, plan, x, mask, pos)
        assert plan.check() == 0, K.last_error()
        for a, n, t in zip(row0, lens, nodes):
            keep[a + n:a + n + t] = False
    torch.cuda.synchronize()
    for a, b in zip(pool.arrays, before.arrays):
        assert torch.equal(a[:, keep], b[:, keep])
