"""GPU: sequences of more drafted rows than a call takes: refused where the host can see it,
else defined: rows behind the most are as rows of no sequence, and are not kept."""
import math

import pytest
import torch

from defer_amd import q8
from test_gpu_draft import random_tree
from test_gpu_q8 import DEV, fill, i32, make_cache, rnd, same, starts

pytestmark = pytest.mark.gpu


def test_more_rows_than_64_a_sequence_want_their_most():
    nh, nkv, hd = 2, 1, 64
    for seqs, rows in ((1, 65), (1, 100), (2, 129), (3, 500)):
        lens = [rows + 20] * seqs
        pages = make_cache(lens, nkv, hd)
        fill(pages, lens, nkv, hd)
        q, tree, kept = rnd(rows, nh, hd, seed=1).to(DEV), i32([-1] * rows), i32([1] * seqs)
        start = i32([0] + [min(rows, 64 * (i + 1)) for i in range(seqs - 1)] + [rows])
        before = [t.clone() for t in pages]
        with pytest.raises(ValueError, match="most_rows"):
            q8.tree_attention(q, pages, tree, i32(lens), start)
        with pytest.raises(ValueError, match="most_rows"):
            q8.kv_keep(pages, i32(lens), start, i32([0] * rows), kept)
        assert all(same(a, b) for a, b in zip(pages, before))
        # rows behind the sequences, in a call that says how many a sequence has
        few = starts([5] * seqs)
        out = q8.tree_attention(q, pages, tree, i32(lens), few, 5)
        assert torch.equal(out[:5 * seqs], q8.tree_attention(q[:5 * seqs], pages, tree[:5 * seqs], i32(lens), few))
        assert not out[5 * seqs:].any()
        assert q8.kv_keep(pages, i32(lens), few, i32([0] * rows), kept, 5).tolist() == [n - 4 for n in lens]
    # as many as there may be, and rows of no sequence at all
    pages = make_cache([70, 64], nkv, hd)
    fill(pages, [70, 64], nkv, hd)
    q = rnd(128, nh, hd, seed=1).to(DEV)
    tree = i32(random_tree(64, 1) * 2)
    args = (q, pages, tree, i32([70, 64]), starts([64, 64]))
    assert torch.equal(q8.tree_attention(*args), q8.tree_attention(*args, 64))
    nobody = pages._replace(table=pages.table[:0])
    assert not q8.tree_attention(q, nobody, tree, i32([]), i32([0])).any()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("history,nh,nkv,hd", [(40, 6, 2, 64), (3, 8, 1, 40), (1500, 4, 2, 64), (700, 4, 1, 128), (90, 2, 2, 256)])
@pytest.mark.parametrize("counts,most", [([100, 10], None), ([7, 3, 0, 30, 5], 5), ([64, 2], 63), ([1, 90, 1], 64)])
def test_rows_behind_the_most_attend_to_nothing(counts, most, history, nh, nkv, hd, dtype):
    lens = [history + n for n in counts]
    pages = make_cache(lens, nkv, hd)
    fill(pages, lens, nkv, hd)
    rows = sum(counts) + 3
    q = rnd(rows, nh, hd, seed=3, dtype=dtype).to(DEV)
    trees = [random_tree(n, n) for n in counts]
    tree = i32(sum(trees, []) + [-1] * 3)
    limit = 64 if most is None else most
    torch.full((rows, nh, hd), math.nan, dtype=dtype, device=DEV)  # what a fresh tensor may hold
    out = q8.tree_attention(q, pages, tree, i32(lens), starts(counts), most)
    into = torch.full((rows, nh, hd), 3.0, dtype=dtype, device=DEV)
    assert q8.tree_attention(q, pages, tree, i32(lens), starts(counts), most, out=into) is into
    at = 0
    for i, n in enumerate(counts):
        m = min(n, limit)
        one = pages._replace(table=pages.table[i:i + 1].contiguous())
        want = q8.tree_attention(q[at:at + m], one, i32(trees[i][:m]), i32([history + m]), starts([m]))
        for got in (out, into):
            assert torch.equal(got[at:at + m], want), i
        assert not out[at + m:at + n].any() and (into[at + m:at + n] == 3).all(), i
        at += n
    assert not out[at:].any() and (into[at:] == 3).all()


def test_rows_behind_the_most_in_calls_of_many_workgroups():
    """Where a wave takes two tiles of rows."""
    seqs, nh, nkv, hd, most = 40, 64, 8, 64, 17
    counts = [(20, 17, 3, 64, 18)[i % 5] for i in range(seqs)]
    assert seqs * nkv * -(-most * nh // nkv // 16) >= 2048
    lens = [50 + n for n in counts]
    pages = make_cache(lens, nkv, hd)
    fill(pages, lens, nkv, hd)
    q = rnd(sum(counts), nh, hd, seed=3).to(DEV)
    trees = [random_tree(n, i) for i, n in enumerate(counts)]
    torch.full_like(q, math.nan)  # what a fresh tensor may hold
    out = q8.tree_attention(q, pages, i32(sum(trees, [])), i32(lens), starts(counts), most)
    at = 0
    for i, n in enumerate(counts):
        m = min(n, most)
        one = pages._replace(table=pages.table[i:i + 1].contiguous())
        want = q8.tree_attention(q[at:at + m], one, i32(trees[i][:m]), i32([50 + m]), starts([m]))
        assert torch.equal(out[at:at + m], want) and not out[at + m:at + n].any(), i
        at += n


@pytest.mark.parametrize("counts,kept,most", [([100, 10], [80, 4], None), ([100, 10], [64, 10], None), ([100, 10], [65, 0], None),
                                              ([9, 2, 0, 7], [7, 2, 3, 6], 5), ([5], [5], 0)])
def test_rows_behind_the_most_are_not_kept(counts, kept, most):
    history, nkv, hd = 50, 2, 64
    lens = [history + n for n in counts]
    pages = make_cache(lens, nkv, hd)
    fill(pages, lens, nkv, hd)
    limit = 64 if most is None else most
    moved = [min(m, n, limit) for m, n in zip(kept, counts)]
    keep = sum(([n - 1 - t for t in range(n)] for n in counts), [])  # backwards: also from behind the most
    old = q8.kv_read(pages, i32(lens), starts(counts), sum(counts), hd)
    got = q8.kv_keep(pages, i32(lens), starts(counts), i32(keep), i32(kept), most)
    assert got.tolist() == [history + m for m in moved]
    new = q8.kv_read(pages, got, starts(moved), sum(moved), hd)
    rows = [sum(counts[:i]) + counts[i] - 1 - t for i, m in enumerate(moved) for t in range(m)]
    for a, b in zip(new, old):
        assert torch.equal(a, b[rows])
    # the rest of the places hold what they held
    rest = [n - m for n, m in zip(counts, moved)]
    after = q8.kv_read(pages, i32(lens), starts(rest), sum(rest), hd)
    rows = [sum(counts[:i]) + counts[i] - m + t for i, m in enumerate(rest) for t in range(m)]
    for a, b in zip(after, old):
        assert torch.equal(a, b[rows])
