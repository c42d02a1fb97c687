"""A move or an acceptance that is refused leaves every pool as it was."""
from __future__ import annotations

import pytest
import torch

from tests.test_pool_move_gpu import bf16_pools, q8_pools

pytestmark = pytest.mark.gpu


def test_refused_moves_leave_the_pools_alone(K, torch_cuda):
    a, other, wide = bf16_pools(2, 300), bf16_pools(65, 300, seed=1), torch.zeros(300, 4096, dtype=torch.int16, device="cuda")
    q8 = q8_pools(2, 300)
    everything = [a, other, wide, *q8]
    before = [t.clone() for t in everything]
    plan = K.PoolMovePlan([200], [0], [100])
    for why, pools in [("overlap", lambda: K.PoolSet.bf16([a[0], a[0]])),
                       ("overlap", lambda: K.PoolSet.bf16([a.view(-1, 576)[:300], a.view(-1, 576)[299:599]])),
                       ("overlap", lambda: K.PoolSet.q8([q8[0][0]], [q8[0][0].view(torch.int32)[:, 0].contiguous().view(
                           torch.float32)], [q8[0][0].view(torch.int16).view(-1)[:300 * 64].view(300, 64)])),
                       ("row 300", lambda: K.PoolSet.bf16([a[0][:299]])),
                       ("row 300", lambda: K.PoolSet.q8(*[t[:, :299].contiguous() for t in q8])),
                       ("at once", lambda: K.PoolSet.bf16(other)),
                       ("0", lambda: K.PoolSet.bf16([])),
                       ("rows of 8192 bytes", lambda: K.PoolSet.bf16([wide], 4032, 64))]:
        with pytest.raises(K.KvlError, match=why):
            plan.move(pools())
    torch.cuda.synchronize()
    assert all(torch.equal(t, b) for t, b in zip(everything, before))


def test_refused_acceptances_leave_the_pools_alone(K, torch_cuda):
    a = bf16_pools(2, 300)
    before = a.clone()
    pools = K.PoolSet.bf16(a)
    base = torch.tensor([10, 60], device="cuda")
    path = torch.tensor([[1, 2, 4], [2, 3, 5]], dtype=torch.int32, device="cuda")
    count = torch.tensor([3, 3], dtype=torch.int32, device="cuda")
    both = torch.tensor([3, 3, 99], dtype=torch.int32, device="cuda")
    for why, args in [("overlaps", (base, path, both[:2], both[1:])), ("overlaps", (base, path, count, path.view(-1)[2:])),
                      ("int32", (base, path.long(), count)), ("contiguous", (base, path[:, ::2], count)),
                      ("contiguous", (base, path.cpu(), count)), ("paths of 1 to 64", (base, path.repeat(1, 22), count)),
                      ("bytes at least", (base, path, count[:1]))]:
        with pytest.raises(K.KvlError, match=why):
            pools.tree_accept(*args)
    torch.cuda.synchronize()
    assert torch.equal(a, before)
    pools.tree_accept(base, path, count)
    assert torch.equal(a[:, 10:13], before[:, [11, 12, 14]]) and torch.equal(a[:, 60:63], before[:, [62, 63, 65]])
