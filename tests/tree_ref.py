"""Plain 64-bit forms of the tree operators and the bounds their results are held to."""
from __future__ import annotations

import numpy as np
import torch

HALF_BF16 = 2.0 ** -8   # half a step of bf16, relative
HALF_F32 = 2.0 ** -24


class Case:
    """A batch of sequences in one pool, with rows of garbage between them."""

    def __init__(self, lens, nodes, q8=False, nh=16, R=512, DR=64, seed=0, hide=0.0, dev="cuda", gap=3, sd=0.7):
        g = torch.Generator(device=dev)
        g.manual_seed(seed)
        r = np.random.RandomState(seed)
        self.lens, self.nodes, self.q8, self.nh, self.R, self.DR = lens, nodes, q8, nh, R, DR
        self.row0, at = [], gap
        for n, t in zip(lens, nodes):
            self.row0.append(at)
            at += n + t + gap
        self.rows = at
        self.total = sum(nodes)
        self.parents = [np.array([-1 if i == 0 or r.rand() < 0.15 else r.randint(0, i) for i in range(t)], np.int32)
                        for t in nodes]
        words = np.zeros(self.total, np.uint64)
        k = 0
        for p in self.parents:
            m = []
            for i, a in enumerate(p):
                m.append((m[a] if a >= 0 else 0) | (1 << i))
            for w in m:
                words[k] = 0 if r.rand() < hide else w
                k += 1
        self.words = words
        self.mask = torch.from_numpy(words.view(np.int64)).to(dev)
        self.q = (torch.randn(self.total, nh, R + DR, device=dev, generator=g) * sd).to(torch.bfloat16)
        if q8:
            self.lat8 = torch.randint(-128, 128, (at, R), device=dev, dtype=torch.int8, generator=g)
            self.lscale = torch.rand(at, device=dev, generator=g) * 0.019 + 0.001
            self.rope = torch.randn(at, DR, device=dev, generator=g).to(torch.bfloat16)
        else:
            self.kv = torch.randn(at, R + DR, device=dev, generator=g).to(torch.bfloat16)
        self.out = torch.full((self.total, nh, R), 7.0, device=dev, dtype=torch.bfloat16)
        self.lse = torch.full((self.total, nh), 7.0, device=dev)
        self.scale = 1.0 / np.sqrt(192.0)

    def seen(self, b, i):
        first = sum(self.nodes[:b])
        w = int(self.words[first + i])
        return list(range(self.lens[b])) + [self.lens[b] + j for j in range(self.nodes[b]) if (w >> j) & 1]

    def rows64(self, b):
        a, n = self.row0[b], self.lens[b] + self.nodes[b]
        if self.q8:
            lat = self.lat8[a:a + n].double() * self.lscale[a:a + n, None].double()
            return lat, self.rope[a:a + n].double()
        return self.kv[a:a + n, :self.R].double(), self.kv[a:a + n, self.R:].double()

    def run(self, plan, stream=0, lse=True, scale=None):
        lse_t = self.lse if lse else None
        scale = self.scale if scale is None else scale
        if self.q8:
            plan.attend_q8(self.out, lse_t, self.q, self.mask, self.lat8, self.lscale, self.rope, self.rows,
                           rope_dim=self.DR, scale=scale, stream=stream)
        else:
            plan.attend_bf16(self.out, lse_t, self.q, self.mask, self.kv, self.rows, rope_dim=self.DR, scale=scale,
                             stream=stream)

    def plan(self, K, **kw):
        return K.TreePlan(self.lens, self.nodes, self.row0, num_heads=self.nh, kv_lora_rank=self.R, **kw)


def check(c: Case, skip=(), scale=None):
    """c.out and c.lse against the formula in 64 bits, node by node.

    A weight p = exp(s - lse) is off by the error of s and lse and by its own
    rounding to bf16, an output element by that times sum p|v| and by its own
    rounding.  ds bounds the error of a score: width + 1 fp32 products and sums
    of magnitude sum |q k| (a tensor core may truncate where a CPU rounds, hence
    the factor 2), and exp2's 2^-22.  The sum of n weights is off by at most
    n half steps of fp32, relative.
    """
    scale = c.scale if scale is None else scale
    first = 0
    for b, t in enumerate(c.nodes):
        lat, rope = c.rows64(b)
        for i in range(t):
            node = first + i
            if node in skip:
                continue
            idx = c.seen(b, i)
            out, lse = c.out[node].double(), c.lse[node].double()
            if not idx:
                assert torch.all(out == 0) and torch.all(torch.isneginf(lse)), (b, i)
                continue
            j = torch.tensor(idx, device=lat.device)
            kl, kr = lat[j], rope[j]
            q = c.q[node].double()
            ql, qr = q[:, :c.R], q[:, c.R:]
            s = (ql @ kl.T + qr @ kr.T) * scale
            want_lse = torch.logsumexp(s, -1)
            p = torch.exp(s - want_lse[:, None])
            want = p @ kl
            size = (ql.abs() @ kl.abs().T + qr.abs() @ kr.abs().T).amax(-1) * abs(scale)
            ds = 2 * (c.R + c.DR + 1) * HALF_F32 * size + 2.0 ** -22
            n = len(idx)
            tol_lse = ds + n * HALF_F32 + 2.0 ** -21 * (1 + want_lse.abs())
            assert torch.all((lse - want_lse).abs() <= tol_lse), (b, i, (lse - want_lse).abs().max().item())
            mass = p @ kl.abs()
            tol = (HALF_BF16 + 3 * ds[:, None] + 2 * n * HALF_F32) * mass * 1.02 + HALF_BF16 * want.abs() * 1.02 + 1e-30
            bad = ((out - want).abs() / tol).max().item()
            assert bad <= 1.0, (b, i, bad)
        first += t
