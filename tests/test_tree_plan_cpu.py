"""The work plan of the tree attention: what it refuses, and that its items cover every batch."""
from __future__ import annotations

import pathlib
import shutil
import subprocess

import numpy as np
import pytest

ROOT = pathlib.Path(__file__).resolve().parents[1]
CSRC = ROOT / "in-c-test_b200" / "csrc"
GROUP, KEYS = 4, 64  # nodes of a group, key rows of a tile


@pytest.fixture(scope="module")
def dump(tmp_path_factory):
    """plans(batches) -> one plan (None: refused) per (lens, nodes, row0, ctas)."""
    nvcc = shutil.which("nvcc")
    if not nvcc:
        pytest.skip("the plan is compiled for the test: no nvcc")
    exe = tmp_path_factory.mktemp("plan") / "tree_plan_dump"
    subprocess.run([nvcc, "-std=c++17", "-O1", f"-I{CSRC}", f"-I{ROOT / 'include'}", "-o", str(exe),
                    str(ROOT / "tests" / "tree_plan_dump.cpp"), str(CSRC / "tree_plan.cu")], check=True)

    def plans(batches):
        text = "".join(f"{len(lens)} {ctas}\n" + "".join(f"{a} {b} {c}\n" for a, b, c in zip(lens, nodes, row0))
                       for lens, nodes, row0, ctas in batches)
        out = subprocess.run([str(exe)], input=text, capture_output=True, text=True, check=True).stdout.split("\n")
        at, got = 0, []
        for _ in batches:
            head = [int(x) for x in out[at].split()]
            at += 1
            if head == [-1]:
                got.append(None)
                continue
            p = dict(zip(("grid", "slots", "max_merge", "rows", "own"), head[:5]))
            n, m = head[5:]
            p["items"] = [dict(zip(("row0", "len", "tree", "node0", "nn", "tile0", "tile1", "slot", "next"),
                                   map(int, x.split()))) for x in out[at:at + n]]
            p["merges"] = [tuple(map(int, x.split())) for x in out[at + n:at + n + m]]
            at += n + m
            got.append(p)
        assert out[at:] == [""]
        return got

    return plans


BAD = [([-1], [1], [0]), ([5], [65], [0]), ([5], [-1], [0]), ([5], [0], [0]), ([5], [1], [-1]),
       ([2 ** 31 - 1], [1], [0]), ([5], [1], [2 ** 31]), ([5], [1], [2 ** 31 - 5]), ([5], [1], [2 ** 63 - 1]),
       ([1, 2], [1, 70], [0, 50]), ([0, 0, 0], [0, 0, 0], [0, 0, 0])]


@pytest.mark.parametrize("lens,nodes,row0", BAD)
def test_refused_before_a_device_is_asked_for(K, lens, nodes, row0):
    with pytest.raises(K.KvlError, match="cached lengths >= 0, 0 to 64 nodes"):
        K.TreePlan(lens, nodes, row0)


def test_refused_batches(dump):
    assert dump([(*b, 148) for b in BAD]) == [None] * len(BAD)


def check_plan(lens, nodes, row0, ctas, p):
    assert 1 <= p["grid"] <= min(ctas, len(p["items"]))
    assert p["rows"] == max(r + n + t for n, t, r in zip(lens, nodes, row0))
    # every item is reached once: CTA c starts with item c
    reached = []
    for c in range(p["grid"]):
        i = c
        while i >= 0:
            reached.append(i)
            assert len(reached) <= len(p["items"])
            i = p["items"][i]["next"]
    assert sorted(reached) == list(range(len(p["items"])))
    # the tiles of every (sequence, group), each once
    by_group = {}
    for i in p["items"]:
        by_group.setdefault(i["node0"], []).append(i)
    merges = {m[0]: m for m in p["merges"]}
    assert len(merges) == len(p["merges"])
    slots, first = [], 0
    for n, t, r in zip(lens, nodes, row0):
        for g in range(0, t, GROUP):
            node0, nn = first + g, min(GROUP, t - g)
            items = sorted(by_group.pop(node0), key=lambda i: i["tile0"])
            at = 0
            for i in items:
                assert (i["row0"], i["len"], i["tree"], i["nn"]) == (r, n, t, nn)
                assert i["tile0"] == at < i["tile1"]
                at = i["tile1"]
            assert at == (n + t + KEYS - 1) // KEYS
            if len(items) == 1:
                assert items[0]["slot"] == -1 and node0 not in merges
                continue
            # partials in the order of the rows, merged in that order
            _, m_nn, m_first, m_count = merges.pop(node0)
            assert m_nn == nn and m_count == len(items) <= p["max_merge"]
            assert [i["slot"] for i in items] == list(range(m_first, m_first + m_count))
            slots += [i["slot"] for i in items]
        first += t
    assert not by_group and not merges
    assert sorted(slots) == list(range(p["slots"]))


def place(r, lens, nodes):
    row0, at = [], int(r.randint(0, 5))
    for n, t in zip(lens, nodes):
        row0.append(at)
        at += n + t + int(r.randint(0, 3))
    return row0


def random_batches(n):
    r = np.random.RandomState(7)
    for k in range(n):
        batch = int(r.choice([1, 2, 3, 8, 20, 64, 200]))
        hi = int(r.choice([3, 70, 300, 5000, 140000])) if batch < 64 else int(r.choice([3, 300, 9000]))
        lens = [int(x) for x in r.randint(0, hi + 1, batch)]
        if r.rand() < 0.4:
            lens = [hi] * batch
        most = int(r.choice([1, 4, 5, 16, 64]))
        nodes = [most] * batch if r.rand() < 0.5 else [int(x) for x in r.randint(0, most + 1, batch)]
        if not sum(nodes):
            nodes[-1] = 1
        yield lens, nodes, place(r, lens, nodes), int(r.choice([1, 2, 3, 7, 16, 147, 148, 148, 148]))


def test_items_cover_every_batch(dump):
    batches = list(random_batches(400))
    for b, p in zip(batches, dump(batches)):
        check_plan(*b, p)


def test_sequences_around_the_tiles(dump):
    lens = [0, 1, 62, 63, 64, 65, 127, 128, 129, 4095, 4096]
    batches = [([n], [t], [3], c) for n in lens for t in (1, 2, 3, 4, 5, 8, 63, 64) for c in (1, 3, 148)]
    batches += [(lens, [t] * len(lens), place(np.random.RandomState(t), lens, [t] * len(lens)), c)
                for t in (1, 4, 5, 64) for c in (1, 2, 5, 148)]
    for b, p in zip(batches, dump(batches)):
        check_plan(*b, p)


def test_longest_sequence_and_largest_grid(dump):
    """Key counts up to the last row below 2^31, and a grid that no list of CTAs could be kept for."""
    batches = [([n], [t], [0], c) for n, t in ((2 ** 31 - 65, 64), (2 ** 31 - 2, 1), (2 ** 31 - 40, 5)) for c in (1, 148)]
    batches += [([700, 20], [5, 1], [0, 800], 2 ** 31 - 1), ([0], [1], [0], 2 ** 31 - 1)]
    for b, p in zip(batches, dump(batches)):
        check_plan(*b, p)


def test_whose_rows_a_sequence_may_append_to(dump):
    """own: no drafted row is another sequence's drafted or cached row, against all pairs."""
    r = np.random.RandomState(8)
    batches = []
    for _ in range(500):
        batch = int(r.randint(1, 6))
        lens = [int(x) for x in r.randint(0, 40, batch)]
        nodes = [int(x) for x in r.randint(0, 9, batch)]
        nodes[int(r.randint(batch))] = 3
        row0 = [int(x) for x in r.randint(0, 120, batch)]
        batches.append((lens, nodes, row0, 148))
    own = [p["own"] for p in dump(batches)]
    for (lens, nodes, row0, _), o in zip(batches, own):
        want = 1
        for a in range(len(lens)):
            mine = set(range(row0[a] + lens[a], row0[a] + lens[a] + nodes[a]))
            for b in range(len(lens)):
                if a != b and mine & set(range(row0[b], row0[b] + lens[b] + nodes[b])):
                    want = 0
        assert o == want, (lens, nodes, row0)
    assert 100 < sum(own) < 400
