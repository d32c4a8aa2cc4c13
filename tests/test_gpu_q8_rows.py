"""GPU: the 8-bit operators on rows of no sequence, wherever in a call they are."""
import pytest
import torch

from defer_amd import q8
from test_gpu_q8 import DEV, fill, i32, make_cache, rnd

pytestmark = pytest.mark.gpu


# one row each, a workgroup's units, units over workgroups, prompts
@pytest.mark.parametrize("lens,counts", [([60, 100], [1, 1]), ([777], [1]), ([3000, 2100], [1, 2]), ([200, 70], [200, 33]), ([2100], [900])])
@pytest.mark.parametrize("nh,nkv,hd", [(6, 2, 64), (8, 2, 128), (3, 1, 40)])
@pytest.mark.parametrize("front,back", [(0, 0), (1, 0), (0, 1), (3, 5), (7, 0), (0, 300), (261, 130)])
def test_attention_rows_of_no_sequence(lens, counts, nh, nkv, hd, front, back):
    pages = make_cache(lens, nkv, hd)
    fill(pages, lens, nkv, hd)
    n = sum(counts)
    q = rnd(front + n + back, nh, hd, seed=5).to(DEV)
    at = [0]
    for c in counts:
        at.append(at[-1] + c)
    want = q8.attention(q[front:front + n].contiguous(), pages, i32(lens), i32(at), max(counts), max(lens))
    args = (i32(lens), i32([front + i for i in at]), max(counts), max(lens))
    junk = torch.full_like(q, float("nan"))  # what a fresh output may hold
    del junk
    out = q8.attention(q, pages, *args)
    assert torch.equal(out[front:front + n], want) and not out[:front].any() and not out[front + n:].any()
    into = torch.full_like(q, 3.0)
    q8.attention(q, pages, *args, out=into)
    assert torch.equal(into[front:front + n], want) and (into[:front] == 3).all() and (into[front + n:] == 3).all()
