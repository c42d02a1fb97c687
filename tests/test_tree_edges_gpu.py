"""Trees and moves where addresses pass 32 bits, where pointers have the least alignment that is allowed, and where
sequences share cached rows."""
from __future__ import annotations

import pytest
import torch

from tests.tree_ref import Case, check

pytestmark = pytest.mark.gpu


def far(c, off, rows):
    """The case's rows at row `off` of a pool of `rows`."""
    names = ("lat8", "lscale", "rope") if c.q8 else ("kv",)
    for name in names:
        t = getattr(c, name)
        big = torch.empty((rows,) + tuple(t.shape[1:]), dtype=t.dtype, device="cuda")
        big[off:off + c.rows] = t
        setattr(c, name, big)
    c.row0 = [r + off for r in c.row0]
    c.rows = rows
    return [getattr(c, name) for name in names]


@pytest.mark.parametrize("q8,rows", [(False, 4_000_000), (True, 8_600_000)], ids=["bf16", "q8"])
@pytest.mark.parametrize("shape", [(16, 512, 64), (3, 512, 64)])
def test_rows_behind_4_gib(K, torch_cuda, q8, rows, shape):
    nh, R, DR = shape
    c = Case([300, 0, 65], [9, 1, 20], q8=q8, nh=nh, R=R, DR=DR, seed=31)
    arrays = far(c, rows - c.rows - 40, rows)
    assert c.row0[0] * (R if q8 else 2 * (R + DR)) > 2 ** 32
    plan = c.plan(K)
    c.run(plan)
    assert plan.check() == 0
    check(c)
    # the path 1, 4, 8 of the first tree is kept, then the sequence goes to the pool's start and back to its end
    pools = K.PoolSet.q8(*[[t] for t in arrays]) if q8 else K.PoolSet.bf16(arrays, R, DR)
    base = c.row0[0] + 300
    want = [t[[base + 1, base + 4, base + 8]].clone() for t in arrays]
    kept = torch.empty(1, dtype=torch.int32, device="cuda")
    pools.tree_accept(torch.tensor([base], device="cuda"), torch.tensor([[1, 4, 8]], dtype=torch.int32, device="cuda"),
                      torch.tensor([3], dtype=torch.int32, device="cuda"), kept)
    assert kept.item() == 3 and all(torch.equal(t[base:base + 3], w) for t, w in zip(arrays, want))
    seq = [t[c.row0[0]:base + 3].clone() for t in arrays]
    K.PoolMovePlan([c.row0[0]], [0], [303]).move(pools)
    assert all(torch.equal(t[:303], w) for t, w in zip(arrays, seq))
    K.PoolMovePlan([0], [rows - 38], [38]).move(pools)
    assert all(torch.equal(t[rows - 38:], w[:38]) for t, w in zip(arrays, seq))
    slide = K.PoolMovePlan([c.row0[0]], [c.row0[0] - 5], [303])
    slide.move(pools)
    assert slide.check() == 0
    assert all(torch.equal(t[c.row0[0] - 5:c.row0[0] + 298], w) for t, w in zip(arrays, seq))


def shifted(t, bytes_):
    """A copy of t that starts `bytes_` behind a 256-byte boundary."""
    flat = torch.empty(t.numel() + 256, dtype=t.dtype, device="cuda")
    at = (-flat.data_ptr() % 256 + bytes_) // t.element_size()
    v = flat[at:at + t.numel()].view(t.shape)
    v.copy_(t)
    assert v.data_ptr() % 256 == bytes_
    return v


@pytest.mark.parametrize("q8", [False, True], ids=["bf16", "q8"])
def test_sixteen_byte_alignment(K, torch_cuda, q8):
    c = Case([700, 3], [13, 6], q8=q8, seed=32)
    for name in ("q", "out") + (("lat8", "rope") if q8 else ("kv",)):
        setattr(c, name, shifted(getattr(c, name), 16))
    c.mask, c.lse = shifted(c.mask, 8), shifted(c.lse, 4)
    if q8:
        c.lscale = shifted(c.lscale, 4)
    c.run(c.plan(K))
    check(c)


@pytest.mark.parametrize("q8", [False, True], ids=["bf16", "q8"])
def test_sequences_that_share_their_cache(K, torch_cuda, q8):
    c = Case([500, 500], [5, 11], q8=q8, seed=33)
    c.row0[1] = c.row0[0]  # the same cached and drafted rows, each under its own masks
    c.run(c.plan(K))
    check(c)


@pytest.mark.parametrize("q8", [False, True], ids=["bf16", "q8"])
def test_negative_and_zero_row_scales(K, torch_cuda, q8):
    c = Case([200, 64], [7, 4], q8=q8, seed=34, hide=0.2)
    if q8:
        c.lscale[::3] *= -1
        c.lscale[5::7] = 0
    c.run(c.plan(K), scale=-0.05)
    check(c, scale=-0.05)


@pytest.mark.parametrize("q8", [False, True], ids=["bf16", "q8"])
@pytest.mark.parametrize("ctas", [1, 2, 5])
@pytest.mark.parametrize("tiles", [[2] * 12, [1] * 9, [3] * 6, [2, 1, 2, 2, 3, 1, 1, 2, 4, 2, 2, 5, 1, 2]])
def test_short_items_follow_one_another(K, torch_cuda, q8, ctas, tiles):
    """A CTA walks many sequences of few tiles: the roles of the kernel are as far apart as they get."""
    lens = [64 * t - 20 for t in tiles]
    c = Case(lens, [4] * len(lens), q8=q8, seed=len(lens) + ctas)
    plan = c.plan(K, max_ctas=ctas)
    for _ in range(5):
        c.out.fill_(3)
        c.run(plan)
        assert plan.check() == 0
    check(c)


def test_plans_serve_other_streams_at_once(K, torch_cuda):
    """Created and used at once on streams that do not wait for the default one, while that one is busy."""
    c = Case([300, 5000], [9, 4], seed=41)
    rows = torch.arange(20000 * 576, device="cuda", dtype=torch.int32).view(20000, 576).to(torch.int16)
    want = rows[100:15100].clone()
    busy = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    for _ in range(5):
        for _ in range(5):
            busy = busy @ busy * 1e-3
        s = torch.cuda.Stream()
        plan = c.plan(K)
        c.run(plan, stream=s.cuda_stream)
        move = K.PoolMovePlan([100], [50], [15000])
        pool = rows.clone()
        s.wait_stream(torch.cuda.current_stream())
        move.move(K.PoolSet.bf16([pool]), stream=s.cuda_stream)
        s.synchronize()
        assert plan.check(s.cuda_stream) == 0 and move.check(s.cuda_stream) == 0
        check(c)
        assert torch.equal(pool[50:15050], want)
        c.out.fill_(3)
        torch.cuda.synchronize()
