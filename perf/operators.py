"""Speculative-decoding operators of the MLA latent cache: what is timed, and their plain forms.

Three operators that a serving loop runs one after the other on a pool of cached rows (576 wide: 512 latent and
64 rope; bf16, or Q8 = int8 latent, fp32 row scale, bf16 rope):

  tree    attention of a tree of drafted tokens over each sequence's cache and over the drafted rows behind it
  accept  the drafted rows that were accepted move up, so that they follow the cached rows (all layers' pools)
  move    runs of rows are copied (a sequence is forked) or slid down (a pool is compacted)

A case is a dict of plain values; `own` chooses between the library's calls and the plain torch forms.
"""
import math
import random

import numpy as np
import torch

own = False

HEADS, RANK, ROPE = 16, 512, 64
WIDTH = RANK + ROPE
SCALE = 1.0 / math.sqrt(192.0)
LAYERS = 27


def listed():
    return [
        # one sequence with a short cache and a small draft: the latency of a call
        {"name": "tree bf16 1x1024 t8", "op": "tree", "q8": False, "batch": 1, "lo": 1024, "hi": 1024, "nodes": 8, "ragged": False},
        # a chat batch of ragged lengths, eight drafted tokens each
        {"name": "tree bf16 64x8192 t8", "op": "tree", "q8": False, "batch": 64, "lo": 512, "hi": 8192, "nodes": 8, "ragged": False},
        # one very long context (split over the whole GPU), a draft that fits one pass over the cache
        {"name": "tree bf16 1x131072 t4", "op": "tree", "q8": False, "batch": 1, "lo": 131072, "hi": 131072, "nodes": 4, "ragged": False},
        # long contexts and wide trees: bound by the tensor cores
        {"name": "tree bf16 16x32768 t64", "op": "tree", "q8": False, "batch": 16, "lo": 32768, "hi": 32768, "nodes": 64, "ragged": False},
        # odd lengths and node counts that differ from sequence to sequence, on the Q8 state
        {"name": "tree q8 5x2777 t13", "op": "tree", "q8": True, "batch": 5, "lo": 1, "hi": 2777, "nodes": 13, "ragged": True},
        # the ragged batch on the Q8 state, a draft that fits one pass over the cache
        {"name": "tree q8 64x8192 t4", "op": "tree", "q8": True, "batch": 64, "lo": 512, "hi": 8192, "nodes": 4, "ragged": False},
        # long contexts on the Q8 state
        {"name": "tree q8 4x32768 t32", "op": "tree", "q8": True, "batch": 4, "lo": 32768, "hi": 32768, "nodes": 32, "ragged": False},
        # after the verification of one layer's pool: a handful of rows
        {"name": "accept bf16 1 pool 1x8", "op": "accept", "q8": False, "pools": 1, "batch": 1, "nodes": 8},
        # after a step of a batch: all layers at once
        {"name": "accept q8 27 pools 64x32", "op": "accept", "q8": True, "pools": LAYERS, "batch": 64, "nodes": 32},
        # a prompt's rows are forked to four continuations in every layer
        {"name": "fork bf16 27 pools 4x4096", "op": "move", "q8": False, "pools": LAYERS, "kind": "fork", "runs": 4, "lo": 4096, "hi": 4096},
        # a layer's pool is compacted after some of its sequences ended
        {"name": "compact bf16 64x8192", "op": "move", "q8": False, "pools": 1, "kind": "compact", "runs": 64, "lo": 512, "hi": 8192},
        # the same on the Q8 state, all layers
        {"name": "compact q8 27 pools 31x1000", "op": "move", "q8": True, "pools": LAYERS, "kind": "compact", "runs": 31, "lo": 1, "hi": 1000},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["tree", "tree", "tree", "accept", "move"])
    q8 = rng.random() < 0.5
    if op == "tree":
        nodes = _log(rng, 1, 64)
        batch = _log(rng, 1, 64)
        most = min(131072, 524288 // batch, 16 * 32768 * 64 // (batch * nodes))
        hi = _log(rng, 1, most)
        lo = rng.choice([0, hi, max(1, hi // 16)])
        return {"op": op, "q8": q8, "batch": batch, "lo": lo, "hi": hi, "nodes": nodes, "ragged": rng.random() < 0.5}
    if op == "accept":
        return {"op": op, "q8": q8, "pools": rng.choice([1, 2, LAYERS]), "batch": _log(rng, 1, 64), "nodes": _log(rng, 2, 64)}
    pools = rng.choice([1, 3, LAYERS])
    runs = _log(rng, 1, 64)
    hi = _log(rng, 1, min(8192, 442368 // (pools * runs)))
    return {"op": op, "q8": q8, "pools": pools, "kind": rng.choice(["fork", "compact"]), "runs": runs,
            "lo": rng.choice([1, hi]), "hi": hi}


# ---------------------------------------------------------------- what a case is made of (its sizes, not its data)
def _rng(case):
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _shape(case):
    """(cached lengths, node counts) of a tree case."""
    r = _rng(case)
    lens = [r.randint(case["lo"], case["hi"]) for _ in range(case["batch"])]
    lens[0] = case["hi"]
    nodes = [r.randint(1, case["nodes"]) if case["ragged"] else case["nodes"] for _ in range(case["batch"])]
    nodes[-1] = case["nodes"]
    return lens, nodes


def _runs(case):
    """(src, dst, count, pool rows) of a move case."""
    r = _rng(case)
    counts = [r.randint(case["lo"], case["hi"]) for _ in range(case["runs"])]
    if case["kind"] == "fork":  # one prompt, forked to `runs` places behind it
        n, src, dst, at = max(counts), [], [], max(counts)
        for c in counts:
            src.append(0)
            dst.append(at)
            at += c + r.randint(0, 64)
        return src, dst, counts, at + 1
    src, dst, at, to = [], [], 0, 0  # sequences that ended leave holes, the others slide down
    for c in counts:
        at += r.choice([0, 0, r.randint(1, max(1, case["hi"]))])
        src.append(at)
        dst.append(to)
        at += c
        to += c
    return src, dst, counts, at + 1


def _tree(r, n):
    """Parents (before their children, -1: a root) of a drafted tree: chains that branch here and there."""
    return [-1 if i == 0 or r.random() < 0.1 else (i - 1 if r.random() < 0.6 else r.randrange(i)) for i in range(n)]


def _masks(parent):
    """Bit j of node i's word: node j is node i or one of its ancestors."""
    m = []
    for i, p in enumerate(parent):
        m.append((m[p] if p >= 0 else 0) | (1 << i))
    return m


# ---------------------------------------------------------------- inputs
def _pool(gen, pools, rows, q8):
    dev = "cuda"
    if not q8:
        return {"kv": torch.randn(pools, rows, WIDTH, device=dev, dtype=torch.bfloat16, generator=gen)}
    return {"lat8": torch.randint(-127, 128, (pools, rows, RANK), device=dev, dtype=torch.int8, generator=gen),
            "scale": torch.rand(pools, rows, device=dev, generator=gen) * 0.019 + 0.001,
            "rope": torch.randn(pools, rows, ROPE, device=dev, dtype=torch.bfloat16, generator=gen)}


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    r = random.Random(seed)
    s = {"case": case}
    if case["op"] == "tree":
        lens, nodes = _shape(case)
        row0, rows = [], 0
        for n, t in zip(lens, nodes):
            row0.append(rows)
            rows += n + t + r.randint(0, 3)
        total = sum(nodes)
        s.update(_pool(gen, 1, rows, case["q8"]))
        s["q"] = (torch.randn(total, HEADS, WIDTH, device="cuda", generator=gen) * 0.7).to(torch.bfloat16)
        words = [w for t in nodes for w in _masks(_tree(r, t))]
        s["mask"] = torch.from_numpy(np.array(words, dtype=np.uint64).view(np.int64)).cuda()
        s["out"] = torch.empty(total, HEADS, RANK, device="cuda", dtype=torch.bfloat16)
        s["lse"] = torch.empty(total, HEADS, device="cuda")
        # sequence and place of every node, for the plain form's padded batch
        s["seq"] = torch.tensor([b for b, t in enumerate(nodes) for _ in range(t)], device="cuda")
        s["at"] = torch.tensor([i for t in nodes for i in range(t)], device="cuda")
        s["row0"] = torch.tensor(row0, device="cuda")
        s["len"] = torch.tensor(lens, device="cuda")
        s["nodes"] = torch.tensor(nodes, device="cuda")
        s["longest"] = max(n + t for n, t in zip(lens, nodes))
        s["widest"] = max(nodes)
        s["rows"] = rows
        if own:
            s["plan"] = _lib().TreePlan(lens, nodes, row0)
    elif case["op"] == "accept":
        t, batch = case["nodes"], case["batch"]
        stride = 192  # rows of a sequence that matter here: the end of its cache and its drafted rows
        rows = batch * stride
        s.update(_pool(gen, case["pools"], rows, case["q8"]))
        path = torch.arange(t).repeat(batch, 1)
        count = []
        for b in range(batch):
            keep = sorted(r.sample(range(t), r.randint(1, max(1, t // 2))))
            path[b, :len(keep)] = torch.tensor(keep)
            count.append(len(keep))
        s["path"] = path.to(torch.int32).cuda()
        s["count"] = torch.tensor(count, dtype=torch.int32, device="cuda")
        s["base"] = torch.tensor([b * stride + r.randint(0, 100) for b in range(batch)], dtype=torch.int64, device="cuda")
        s["kept"] = torch.empty(batch, dtype=torch.int32, device="cuda")
        s["rows"] = rows
        if own:
            s["pools"] = _lib().PoolSet.q8(s["lat8"], s["scale"], s["rope"]) if case["q8"] else _lib().PoolSet.bf16(s["kv"])
    else:
        src, dst, count, rows = _runs(case)
        s.update(_pool(gen, case["pools"], rows, case["q8"]))
        s["from"] = torch.cat([torch.arange(a, a + n) for a, n in zip(src, count)]).cuda()
        s["to"] = torch.cat([torch.arange(a, a + n) for a, n in zip(dst, count)]).cuda()
        if own:
            s["pools"] = _lib().PoolSet.q8(s["lat8"], s["scale"], s["rope"]) if case["q8"] else _lib().PoolSet.bf16(s["kv"])
            s["plan"] = _lib().PoolMovePlan(src, dst, count)
    return s


def _lib():
    import kvl_pkg
    kvl_pkg.load()
    import kvl_b200.kvl_mla as K
    return K


# ---------------------------------------------------------------- one pass
def _bits(s):
    """The pool as whole numbers: a copied row is the same row bit for bit."""
    if "kv" in s:
        return [s["kv"].view(torch.int16)]
    return [s["lat8"], s["scale"].view(torch.int32), s["rope"].view(torch.int16)]


def _plain_tree(s):
    b, k = s["row0"].numel(), s["longest"]
    places = torch.arange(k, device="cuda")
    at = (s["row0"][:, None] + places).clamp_(max=s["rows"] - 1)
    if s["case"]["q8"]:
        kv = torch.cat([s["lat8"][0][at].float() * s["scale"][0][at][..., None], s["rope"][0][at].float()], -1)
    else:
        kv = s["kv"][0][at].float()
    q = torch.zeros(b, s["widest"], HEADS, WIDTH, device="cuda")
    q[s["seq"], s["at"]] = s["q"].float()
    word = torch.zeros(b, s["widest"], device="cuda", dtype=torch.int64)
    word[s["seq"], s["at"]] = s["mask"]
    node = places - s["len"][:, None]                                   # [b][k] number of the drafted row
    bit = (word[:, :, None] >> node.clamp(0, 63)[:, None]) & 1
    drafted = (node >= 0) & (node < s["nodes"][:, None])
    seen = (node < 0)[:, None] | (drafted[:, None] & (bit == 1))        # [b][nodes][k]
    x = torch.matmul(q.reshape(b, -1, WIDTH), kv.transpose(1, 2)).mul_(SCALE).view(b, -1, HEADS, k)
    x.masked_fill_(~seen[:, :, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    x = x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(b, -1, k), kv[..., :RANK]).view(b, -1, HEADS, RANK)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    lse = (top + total.log()).squeeze(-1)
    return o[s["seq"], s["at"]].to(torch.bfloat16), lse[s["seq"], s["at"]]


def run(state):
    s, case = state, state["case"]
    if case["op"] == "tree":
        if own:
            if case["q8"]:
                s["plan"].attend_q8(s["out"], s["lse"], s["q"], s["mask"], s["lat8"], s["scale"], s["rope"], s["rows"])
            else:
                s["plan"].attend_bf16(s["out"], s["lse"], s["q"], s["mask"], s["kv"], s["rows"])
            return {"out": s["out"], "lse": s["lse"]}
        out, lse = _plain_tree(s)
        return {"out": out, "lse": lse}
    if case["op"] == "accept":
        if own:
            s["pools"].tree_accept(s["base"], s["path"], s["count"], s["kept"])
            return {"pool": _bits(s), "kept": s["kept"]}
        j = torch.arange(case["nodes"], device="cuda")
        source = s["base"][:, None] + torch.where(j < s["count"][:, None], s["path"].long(), j)
        dest = s["base"][:, None] + j
        for t in _bits(s):
            t[:, dest] = t[:, source]
        return {"pool": _bits(s), "kept": s["count"].clone()}
    if own:
        s["plan"].move(s["pools"])
    else:
        for t in _bits(s):
            t[:, s["to"]] = t[:, s["from"]]
    return {"pool": _bits(s)}


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    row = RANK + 4 + 2 * ROPE if case["q8"] else 2 * WIDTH
    if case["op"] == "tree":
        lens, nodes = _shape(case)
        total = sum(nodes)
        pairs = sum(n * t + t for n, t in zip(lens, nodes))
        return {"bytes": row * (sum(lens) + total) + total * (HEADS * (2 * WIDTH + 2 * RANK + 4) + 8),
                "flops": 2 * HEADS * (WIDTH + RANK) * pairs}
    if case["op"] == "accept":
        moved = case["batch"] * max(1, case["nodes"] // 4)  # about that many of the drafted rows are kept
        return {"bytes": 2 * case["pools"] * moved * row + case["batch"] * (4 * case["nodes"] + 16), "flops": 0}
    src, dst, count, _ = _runs(case)
    if case["kind"] == "fork":
        return {"bytes": case["pools"] * row * (sum(count) + max(count)), "flops": 0}
    moved = sum(n for a, b, n in zip(src, dst, count) if a != b)
    return {"bytes": max(row, 2 * case["pools"] * row * moved), "flops": 0}


# ---------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    if case["op"] != "tree":
        return None  # copies: nothing is computed
    s = prepare(case, seed)
    lens, nodes = _shape(case)
    row0 = s["row0"].tolist()
    words = s["mask"].cpu().numpy().view(np.uint64)
    outs, lses, first = [], [], 0
    for n, t, a in zip(lens, nodes, row0):
        if case["q8"]:
            latent = s["lat8"][0, a:a + n + t].double() * s["scale"][0, a:a + n + t, None].double()
            rope = s["rope"][0, a:a + n + t].double()
        else:
            latent, rope = s["kv"][0, a:a + n + t].double().split([RANK, ROPE], -1)
        see = np.ones((t, n + t), bool)
        for i in range(t):
            for j in range(t):
                see[i, n + j] = (int(words[first + i]) >> j) & 1
        see = torch.from_numpy(see).cuda()
        for i in range(0, t, 8):  # eight nodes at a time, for the memory's sake
            q = s["q"][first + i:first + min(i + 8, t)].double()
            x = (torch.einsum("thd,kd->thk", q[..., :RANK], latent) + torch.einsum("thd,kd->thk", q[..., RANK:], rope)) * SCALE
            x = x.masked_fill(~see[i:i + 8, None], -math.inf)
            lse = torch.logsumexp(x, -1)
            w = torch.exp(x - torch.where(lse == -math.inf, 0.0, lse)[..., None])
            outs.append(torch.einsum("thk,kd->thd", w, latent))
            lses.append(lse)
        first += t
    return {"out": torch.cat(outs), "lse": torch.cat(lses)}
