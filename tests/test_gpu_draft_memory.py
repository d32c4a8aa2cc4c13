"""GPU: a verifying step, captured and replayed or on two streams, writes nothing but what is its own: patterns in
memory that the program holds beside it, and allocates between the replays, stay as they are."""
import torch

import pytest

from defer_amd import q8
from test_gpu_draft import random_tree
from test_gpu_q8 import DEV, fill, i32, make_cache, rnd, same, starts

pytestmark = pytest.mark.gpu


class Patterns:
    """Tensors of sizes that the step's own have, each filled with a number of its own."""
    SIZES = (1, 29, 4096, 29 * 8 * 64, 1 << 18, 3 << 20)

    def __init__(self):
        self.held = []

    def more(self):
        for n in self.SIZES:
            self.held.append((len(self.held) + 1, torch.full((n,), len(self.held) + 1, dtype=torch.int32, device=DEV)))

    def whole(self):
        return all(bool((t == v).all()) for v, t in self.held)


def case():
    nh, nkv, hd, lens, counts = 8, 2, 64, [1900, 800], [9, 20]
    history = make_cache(lens, nkv, hd)
    fill(history, lens, nkv, hd)
    tree = i32(random_tree(9, 1) + random_tree(20, 2))
    q, k, v = (rnd(29, h, hd, seed=i).to(DEV) for i, h in enumerate((nh, nkv, nkv)))
    logits, rot = rnd(29, 50000, seed=5).to(DEV), q8.rotary(hd, device=DEV)
    target, kv_len, start = i32(list(range(29))), i32(lens), starts(counts)
    keep, kept = i32([0, 2, 4] + [-1] * 6 + [1, 5, 7, 19] + [-1] * 16), i32([3, 4])

    def step(pages):
        a = q8.kv_append(pages, q, k, v, kv_len, rot, start, 20)
        o = q8.tree_attention(a, pages, tree, kv_len, start, 20, 1900)
        return (a, o) + tuple(q8.log_probs(logits, target, 20)) + (q8.kv_keep(pages, kv_len, start, keep, kept, 20),)

    def fresh():
        return q8.Pages(*[t.clone() for t in history[:4]], history.table)

    return step, fresh


def test_replays_write_nothing_else():
    step, fresh = case()
    want_pages = fresh()
    want = step(want_pages)
    beside = Patterns()
    beside.more()
    pages, start = fresh(), fresh()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(pages)
    beside.more()
    for _ in range(4):
        for a, b in zip(pages[:4], start[:4]):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(same(a, b) for a, b in zip(got, want)) and all(same(a, b) for a, b in zip(pages, want_pages))
        assert beside.whole()
        own = fresh()
        assert all(same(a, b) for a, b in zip(step(own), want)) and beside.whole()
        beside.more()


def test_steps_on_two_streams_write_nothing_else():
    step, fresh = case()
    want_pages = fresh()
    want = step(want_pages)
    beside = Patterns()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        beside.more()
        pages = [fresh() for _ in streams]
        torch.cuda.synchronize()
        got = []
        for s, p in zip(streams, pages):
            with torch.cuda.stream(s):
                got.append(step(p))
        torch.cuda.synchronize()
        for g, p in zip(got, pages):
            assert all(same(a, b) for a, b in zip(g, want)) and all(same(a, b) for a, b in zip(p, want_pages))
        assert beside.whole()
