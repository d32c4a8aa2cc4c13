"""GPU: the attention of trees over histories long enough that a row's units are dealt to workgroups and
joined: every head size and type, hidden places, pages that are not there, rows of no sequence."""
import pytest
import torch

from defer_amd import q8
from test_gpu_draft import check_tree, random_tree
from test_gpu_q8 import DEV, TYPES, fill, i32, make_cache, rnd, starts

pytestmark = pytest.mark.gpu
SIZES = [(6, 2, 64), (8, 1, 128), (4, 2, 192), (5, 1, 160), (4, 1, 256), (3, 3, 200)]


def dealt(pages, counts, heads, most_len):
    """Whether these rows are dealt, by the size of the workspace that they want."""
    p = q8._CPages(*[None] * 5, 1, pages.keys.shape[1], pages.keys.shape[3], 1)
    r = q8._CRows(None, None, len(counts), sum(counts), max(counts))
    return q8._lib().defer_gpu_q8_tree_attention_workspace(p, r, heads, most_len) > 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nh,nkv,hd", SIZES)
def test_dealt_rows_have_their_paths_bits(nh, nkv, hd, dtype):
    ctxs, trees = [390, 700, 511, 0, 1500], [random_tree(n, n) for n in (6, 11, 5, 7, 17)]
    h = torch.rand(5, 1510, generator=torch.Generator().manual_seed(hd)) < 0.3
    h[1] = True             # sees nothing
    h[4, :1400] = True      # nothing of most units
    for hidden in (None, h):
        out = check_tree(ctxs, trees, nh, nkv, hd, dtype=dtype, hidden=hidden, seed=hd, some=[0, 2, 4], formula=hidden is None)
        assert dealt(out[1], out[4], nh, max(out[3]))
        assert hidden is None or not out[-1][6:17].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nh,nkv,hd", SIZES)
def test_dealt_rows_beside_rows_of_no_sequence_and_pages_that_are_not_there(nh, nkv, hd, dtype):
    counts, ctxs = [9, 4], [640, 1100]
    lens = [c + n for c, n in zip(ctxs, counts)]
    pages = make_cache(lens, nkv, hd, seed=1)
    fill(pages, lens, nkv, hd, seed=1)
    assert dealt(pages, counts, nh, max(lens))
    q = rnd(18, nh, hd, seed=2, dtype=dtype).to(DEV)
    tree = i32([-1, -1] + random_tree(9, 1) + random_tree(4, 2) + [-1] * 3)
    start = i32([2, 11, 15])
    plain = q8.tree_attention(q[2:15], pages, tree[2:15].contiguous(), i32(lens), starts(counts), 9, max(lens))
    out = q8.tree_attention(q, pages, tree, i32(lens), start, 9, max(lens))
    assert torch.equal(out[2:15], plain) and not out[:2].any() and not out[15:].any()
    into = torch.full_like(q, 3.0)
    q8.tree_attention(q, pages, tree, i32(lens), start, 9, max(lens), out=into)
    assert torch.equal(into[2:15], plain) and (into[:2] == 3).all() and (into[15:] == 3).all()
    own = q.clone()
    assert torch.equal(q8.tree_attention(own, pages, tree, i32(lens), start, 9, max(lens), out=own)[2:15], plain)
    # pages of the history and of drafted rows: as if what they held were hidden
    for gone in ((0,), (3, 4), (10,), (17,), tuple(range(18))):
        table, h = pages.table.clone(), torch.zeros(2, 1152, dtype=torch.uint8, device=DEV)
        for p in gone:
            h[:, 64 * p:64 * p + 64] = 1
            table[:, p:p + 1] = -1
        a = q8.tree_attention(q, pages._replace(table=table), tree, i32(lens), start, 9, max(lens))
        assert torch.equal(a, q8.tree_attention(q, pages, tree, i32(lens), start, 9, max(lens), hidden=h)), gone
        assert len(gone) < 18 or not a.any()
