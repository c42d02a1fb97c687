"""What the tree and move calls refuse before they touch a device."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest


def test_tree_mask(K):
    m = K.tree_mask([-1, 0, 0, 1, -1, 3])
    assert [int(x) for x in m] == [1, 3, 5, 11, 16, 43]
    chain = K.tree_mask(list(range(-1, 63)))
    assert [int(x) for x in chain] == [(1 << (i + 1)) - 1 for i in range(64)]
    for bad in ([0], [-2], [-1, 1], [-1, 0, 5], list(range(-1, 64)), []):
        with pytest.raises(K.KvlError):
            K.tree_mask(bad)


@pytest.mark.parametrize("lens,nodes,row0", [([-1], [1], [0]), ([5], [65], [0]), ([5], [-1], [0]), ([5], [0], [0]),
                                             ([5], [1], [-1]), ([2 ** 31 - 1], [1], [0]), ([5], [1], [2 ** 31]),
                                             ([5], [1], [2 ** 31 - 5]), ([], [], []), ([1, 2], [1], [0])])
def test_tree_plan_refusals(K, lens, nodes, row0):
    with pytest.raises(K.KvlError):
        K.TreePlan(lens, nodes, row0)


def test_tree_plan_null_arguments(K):
    lib = K.load()
    h = C.c_void_p()
    one = np.array([1], np.int32)
    r0 = np.array([0], np.int64)
    p, q = K.ptr(one, K.i32p), K.ptr(r0, K.i64p)
    assert lib.kvl_mla_tree_plan_create(None, 1, p, p, q, 16, 512, 0) == -1
    assert lib.kvl_mla_tree_plan_create(C.byref(h), 1, None, p, q, 16, 512, 0) == -1
    assert lib.kvl_mla_tree_plan_create(C.byref(h), 1, p, None, q, 16, 512, 0) == -1
    assert lib.kvl_mla_tree_plan_create(C.byref(h), 1, p, p, None, 16, 512, 0) == -1
    assert lib.kvl_mla_tree_plan_create(C.byref(h), 1, p, p, q, 0, 512, 0) == -1
    assert lib.kvl_mla_tree_plan_create(C.byref(h), 1, p, p, q, 16, 0, 0) == -1
    assert lib.kvl_mla_tree_plan_create(C.byref(h), 1, p, p, q, 16, 512, -1) == -1
    assert not h
    lib.kvl_mla_tree_plan_destroy(None)
    assert lib.kvl_mla_tree_plan_info(None, None, None, None) == -1
    assert lib.kvl_mla_tree_check(None, None) == -1


@pytest.mark.parametrize("src,dst,count,why", [
    ([-1], [0], [1], "range"), ([0], [-1], [1], "range"), ([0], [1], [-1], "range"), ([2 ** 31], [0], [1], "range"),
    ([0], [2 ** 31 - 2], [5], "range"),
    ([0, 100], [200, 209], [10, 10], "write row"),
    ([0, 100], [200, 200], [10, 10], "write row"),
    ([0], [5], [10], "reads"),                 # up, onto itself
    ([0, 100], [100, 0], [50, 50], "reads"),   # a swap
    ([100, 70], [30, 60], [30, 20], "reads"),  # down, but the runs cross
    ([50, 60], [0, 55], [20, 20], "reads"),    # sources overlap
    ([10, 30], [0, 40], [10, 20], "reads"),    # one of them up
])
def test_move_plan_refusals(K, src, dst, count, why):
    with pytest.raises(K.KvlError, match=why):
        K.PoolMovePlan(src, dst, count)


def test_null_arguments_of_moves(K):
    lib = K.load()
    assert lib.kvl_mla_move_plan_create(None, 1, None, None, None) == -1
    h = C.c_void_p()
    assert lib.kvl_mla_move_plan_create(C.byref(h), 1, None, None, None) == -1
    assert lib.kvl_mla_move_plan_create(C.byref(h), 0, None, None, None) == -1
    lib.kvl_mla_move_plan_destroy(None)
    assert lib.kvl_mla_move_plan_info(None, None, None) == -1
    assert lib.kvl_mla_move_check(None, None) == -1
    assert lib.kvl_mla_pool_move_bf16(None, None, 1, 10, 512, 64, None) == -1
    assert lib.kvl_mla_pool_move_q8(None, None, None, None, 1, 10, 512, 64, None) == -1
    pools = (C.c_void_p * 2)(4096, 0)
    one = (C.c_void_p * 1)(4096)
    fn = lib.kvl_mla_tree_accept_bf16
    for args in [(None, 1, 10, 512, 64, 1, 8, 8, 8, 4, None, None), (pools, 2, 10, 512, 64, 1, 8, 8, 8, 4, None, None),
                 (one, 0, 10, 512, 64, 1, 8, 8, 8, 4, None, None), (one, 1, 0, 512, 64, 1, 8, 8, 8, 4, None, None),
                 (one, 1, 10, 0, 64, 1, 8, 8, 8, 4, None, None), (one, 1, 10, 512, 64, 0, 8, 8, 8, 4, None, None),
                 (one, 1, 10, 512, 64, 1, None, 8, 8, 4, None, None), (one, 1, 10, 512, 64, 1, 8, None, 8, 4, None, None),
                 (one, 1, 10, 512, 64, 1, 8, 8, None, 4, None, None), (one, 1, 10, 512, 64, 1, 8, 8, 8, 0, None, None),
                 (one, 1, 10, 512, 64, 1, 8, 8, 8, 65, None, None), (one, 1, 10, 512, 64, 1, 4, 8, 8, 4, None, None),
                 (one, 1, 10, 512, 64, 1, 8, 64, 96, 4, 96, None), (one, 1, 10, 512, 64, 1, 8, 64, 96, 4, 12, None),
                 (one, 1, 10, 512, 64, 1, 8, 64, 96, 4, 76, None)]:
        assert fn(*args) == -1, args
