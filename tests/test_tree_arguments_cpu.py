"""What the wrappers of the tree and move calls refuse before they hand bare pointers to the library: tensors that are
not on a GPU, not contiguous, too short or of another width.  The library and the GPU are stood in for."""
from __future__ import annotations

import pytest
import torch


class Gpu:
    """A tensor that says that it is on a GPU."""

    def __init__(self, t):
        self.t = t
        self.is_cuda = True

    def __getattr__(self, name):
        return getattr(self.t, name)

    def __iter__(self):
        return (Gpu(t) for t in self.t)


def gpu(*shape, dtype=torch.bfloat16):
    return Gpu(torch.zeros(*shape, dtype=dtype))


class Library:
    """Takes every call and notes it."""

    def __init__(self, K):
        self.K, self.calls = K, []

    def __getattr__(self, name):
        def call(*args):
            if name == "kvl_mla_decode_step_workspace_bytes":
                return self.K.load().kvl_mla_decode_step_workspace_bytes(*args)
            self.calls.append(name)
            return 0
        return call


NODES, ROWS = 3, 50


@pytest.fixture
def plan(K):
    return K.TreePlan([20, 10], [2, 1], [0, 30], lib=Library(K))


def attend_args(q8):
    a = dict(out=gpu(NODES, 16, 512), lse=gpu(NODES, 16, dtype=torch.float32), q=gpu(NODES, 16, 576),
             mask=gpu(NODES, dtype=torch.int64), rows=ROWS)
    a.update(dict(lat8=gpu(ROWS, 512, dtype=torch.int8), lscale=gpu(ROWS, dtype=torch.float32), rope16=gpu(ROWS, 64))
             if q8 else dict(kv=gpu(ROWS, 576)))
    return a


def step_args(K, q8):
    cfg = K.make_config(256, 16, 128, 64, 128, 512, 1e-5, 50000.0)
    size = K.load().kvl_mla_decode_step_workspace_bytes(cfg, NODES)
    a = dict(cfg=cfg, weights=K.KvlMlaDeviceWeights(), out=gpu(NODES, 256, dtype=torch.float32),
             x=gpu(NODES, 256, dtype=torch.float32), mask=gpu(NODES, dtype=torch.int64), pos=gpu(NODES, dtype=torch.int32),
             workspace=gpu(size, dtype=torch.uint8), rows=ROWS)
    a.update({k: v for k, v in attend_args(q8).items() if k in ("kv", "lat8", "lscale", "rope16")})
    return a


def spoilt(t):
    """The same tensor on the host, with a step between its elements, spread without memory, and one element short."""
    yield t.t
    yield Gpu(torch.zeros([2 * n for n in t.shape], dtype=t.dtype)[tuple(slice(None, None, 2) for _ in t.shape)])
    yield Gpu(torch.zeros(1, dtype=t.dtype).expand(t.shape))
    yield Gpu(t.t.flatten()[:-1])


@pytest.mark.parametrize("q8", [False, True], ids=["bf16", "q8"])
@pytest.mark.parametrize("call", ["attend", "step"])
def test_attend_and_step(K, plan, call, q8):
    args = attend_args(q8) if call == "attend" else step_args(K, q8)
    fn = getattr(plan, f"{call}_{'q8' if q8 else 'bf16'}")
    fn(**args)
    assert plan.lib.calls[1:] == [f"kvl_mla_tree_{call}_{'q8' if q8 else 'bf16'}"]
    if call == "attend":
        fn(**{**args, "lse": None})
    seen = len(plan.lib.calls)
    for name, t in args.items():
        if not isinstance(t, Gpu):
            continue
        for k, bad in enumerate(spoilt(t)):
            if k == 3 and call == "step" and name in ("mask", "pos"):
                continue  # the plan's own faults come first
            with pytest.raises(K.KvlError, match=f"{name} must be contiguous"):
                fn(**{**args, name: bad})
    with pytest.raises(K.KvlError, match="must be contiguous"):
        fn(**{**args, "rows": ROWS + 1})
    assert len(plan.lib.calls) == seen


def test_accept(K):
    pools = K.PoolSet.bf16(gpu(2, 10, 576), lib=Library(K))
    good = dict(base=gpu(2, dtype=torch.int64), path=gpu(2, 4, dtype=torch.int32), count=gpu(2, dtype=torch.int32),
                kept=gpu(2, dtype=torch.int32))
    pools.tree_accept(**good)
    pools.tree_accept(**{**good, "kept": None})
    calls = len(pools.lib.calls)
    assert calls == 2
    for name in good:
        for bad in list(spoilt(good[name]))[:3]:
            with pytest.raises(K.KvlError, match=f"{name} must be contiguous"):
                pools.tree_accept(**{**good, name: bad})
        if name in ("path", "count"):
            with pytest.raises(K.KvlError, match="path and count are int32"):
                pools.tree_accept(**{**good, name: gpu(*good[name].shape, dtype=torch.int64)})
    with pytest.raises(K.KvlError, match="base must be"):
        pools.tree_accept(**{**good, "base": gpu(2, dtype=torch.int32)})
    for name in ("count", "kept"):
        with pytest.raises(K.KvlError, match=name):
            pools.tree_accept(**{**good, name: gpu(1, dtype=torch.int32)})
    with pytest.raises(K.KvlError, match="path must be"):
        pools.tree_accept(**{**good, "path": gpu(1, 4, dtype=torch.int32)})
    assert len(pools.lib.calls) == calls


def test_pools_on_the_host(K):
    with pytest.raises(K.KvlError, match="on a GPU"):
        K.PoolSet.bf16(torch.zeros(2, 10, 576, dtype=torch.bfloat16), lib=Library(K))
    with pytest.raises(K.KvlError, match="on a GPU"):
        K.PoolSet.q8(gpu(1, 10, 512, dtype=torch.int8), torch.zeros(1, 10), gpu(1, 10, 64), lib=Library(K))
