"""GPU: the operators that verify drafted tokens (defer_amd.q8: kv_append, tree_attention, kv_keep,
log_probs) against plain 64-bit implementations on the CPU, and against the operators
whose bits they promise."""
import math
from fractions import Fraction

import numpy as np
import pytest
import torch

from defer_amd import q8
from test_gpu_q8 import (DEV, HALF, TYPES, fill, i8, i32, make_cache, ref_attention, ref_codes, rnd, same, starts, tolerance,
                         values)

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ append

PI = Fraction(31415926535897932384626433832795028841971693993751058209749445923, 10 ** 64)


def angles(pos, freq):
    """Positions times frequencies, less the whole turns."""
    per = [Fraction(f) / (2 * PI) for f in freq.tolist()]
    turns = [[float((p * f) % 1) for f in per] for p in pos.tolist()]
    return 2 * math.pi * torch.tensor(turns, dtype=torch.float64).view(len(pos), len(freq))


def turned(x, weight, eps, freq, interleaved, factor, pos):
    """Heads normed and turned, 64 bits."""
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + float(np.float32(eps))) * weight.double()
    n = 2 * len(freq)
    a = angles(pos, freq)[:, None]
    c, s = torch.cos(a) * factor, torch.sin(a) * factor
    i, j = (slice(0, n, 2), slice(1, n, 2)) if interleaved else (slice(0, n // 2), slice(n // 2, n))
    out = x.clone()
    out[..., i] = x[..., i] * c - x[..., j] * s
    out[..., j] = x[..., j] * c + x[..., i] * s
    return out


def check_append(lens, counts, nh, nkv, hd, rotated, interleaved=False, norm=False, dtype=torch.float32, position=None, seed=0,
                 theta=10000.0, factor=1.0, rows=None, scale=1.0):
    rows = sum(counts) if rows is None else rows
    pages = make_cache(lens, nkv, hd, seed=seed)
    q, k, v = (rnd(rows, h, hd, seed=seed + i, dtype=dtype, scale=scale) for i, h in enumerate((nh, nkv, nkv)))
    qn, kn = ((1 + rnd(hd, seed=seed + 5 + i) / 4).to(dtype) for i in range(2)) if norm else (None, None)
    rot = q8.rotary(rotated, theta, interleaved=interleaved, factor=factor, device=DEV)
    gpu = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    out = q8.kv_append(pages, gpu(q), gpu(k), gpu(v), i32(lens), rot, starts(counts), max(counts), position=gpu(position),
                       q_norm=gpu(qn), k_norm=gpu(kn), eps=1e-5)
    pos = torch.cat([torch.arange(n - c, n) for n, c in zip(lens, counts)]) if position is None else position
    used = sum(counts)
    freq = rot.freq.cpu()
    want = turned(q[:used], qn, 1e-5, freq, interleaved, factor, pos[:used])
    assert out.dtype == dtype and out.shape == q.shape
    # half a step of the type, and of f32 before it; 64-bit roundings of what cancels
    tol = (HALF[dtype] + HALF[torch.float32]) * 1.01 * want.abs() + 1e-11 * scale + (2.0 ** -25 if dtype == torch.float16 else 0)
    assert ((out[:used].cpu().double() - want).abs() <= tol).all()
    assert not out[used:].any()
    kc, ks, off = ref_codes(turned(k[:used], kn, 1e-5, freq, interleaved, factor, pos[:used]))
    vc, vs, _ = ref_codes(v[:used].double())
    at = 0
    table = pages.table.cpu()
    for i, (n, c) in enumerate(zip(lens, counts)):
        for j in range(c):
            t = n - c + j
            if t < 0:
                continue
            page, place = int(table[i, t // 64]), t % 64
            got = pages.keys[page, :, place, :hd].cpu()
            assert ((got == kc[at + j]) | (off[at + j] < 1e-6)).all() and (got.int() - kc[at + j].int()).abs().max() <= 1
            assert torch.allclose(pages.key_scale[page, :, place].cpu(), ks[at + j], rtol=2.0 ** -23, atol=0)
            assert torch.equal(pages.values[page, :, :hd, place].cpu(), vc[at + j])
            assert torch.equal(pages.value_scale[page, :, place].cpu(), vs[at + j])
        at += c
    return pages


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nh,nkv,hd,rotated,interleaved,norm", [
    (9, 3, 64, 64, False, False), (8, 2, 128, 128, False, True), (4, 2, 16, 8, True, False), (3, 3, 40, 20, False, True),
    (5, 1, 64, 16, True, True), (6, 2, 80, 80, False, True), (2, 1, 1, 0, False, True), (10, 1, 200, 100, True, True),
    (4, 1, 256, 256, False, True), (4, 2, 100, 50, False, False), (2, 2, 7, 6, True, True), (48, 1, 96, 48, False, True),
    (3, 1, 256, 64, False, False), (2, 1, 192, 192, False, True)])
def test_append(nh, nkv, hd, rotated, interleaved, norm, dtype):
    check_append([1, 63, 64, 65, 200, 7, 130], [1, 63, 3, 0, 50, 7, 17], nh, nkv, hd, rotated, interleaved, norm, dtype, seed=hd)
    check_append([5, 64, 300], [1, 1, 1], nh, nkv, hd, rotated, interleaved, norm, dtype, seed=hd + 1)


def test_append_far_positions_factors_and_frequencies():
    pos = torch.tensor([0, 1, 2 ** 20, 2 ** 24 + 1, 123456789, -5, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32)
    check_append([20], [5], 4, 2, 64, 64, position=pos[:5], factor=1.25)
    check_append([20], [6], 2, 1, 128, 64, True, position=pos[:6], theta=5e5, norm=True, factor=-0.5)
    q, k = rnd(8, 2, 64, seed=1), rnd(8, 1, 64, seed=2)
    pages = make_cache([8], 1, 64)
    rot = q8.rotary(64, 1e4, device=DEV)
    out = q8.kv_append(pages, q.to(DEV), k.to(DEV), k.to(DEV), i32([8]), rot, starts([8]), 8, position=pos.to(DEV))
    want = turned(q, None, 0, rot.freq.cpu(), False, 1.0, pos)
    assert ((out.cpu().double() - want).abs() <= 2.02 * HALF[torch.float32] * want.abs() + 1e-11).all()
    for kw in (dict(scale=4.0), dict(scale=8.0, original_len=8192), dict(scale=8.0, original_len=1000, low=0.5, high=32)):
        f = q8.rotary(64, 5e5, device="cpu", **kw).freq
        plain = q8.rotary(64, 5e5, device="cpu").freq
        assert f.dtype == torch.float64 and (f <= plain).all() and (f >= plain / kw["scale"] * (1 - 1e-12)).all()
        if "original_len" not in kw:
            assert torch.equal(f, plain / 4)
        else:
            assert f[0] == plain[0] and abs(f[-1] / plain[-1] - 1 / 8) < 1e-12 and (f[1:] < f[:-1]).all()


def test_append_without_rotation_is_the_cache_write():
    lens, counts = [70, 3, 130], [40, 3, 1]
    for dtype in TYPES:
        for hd in (64, 72, 200):
            q, k, v = (rnd(44, h, hd, seed=i, dtype=dtype).to(DEV) for i, h in enumerate((4, 2, 2)))
            a, b = make_cache(lens, 2, hd, seed=1), make_cache(lens, 2, hd, seed=1)
            b.keys.copy_(a.keys)
            b.values.copy_(a.values)
            out = q8.kv_append(a, q, k, v, i32(lens), q8.rotary(0, device=DEV), starts(counts), 40)
            q8.kv_write(b, k, v, i32(lens), starts(counts), 40)
            assert torch.equal(out, q) and all(same(x, y) for x, y in zip(a, b))


def test_append_strides_alignments_and_calls_give_the_same_bits():
    nh, nkv, hd, n = 6, 2, 64, 150
    rot = q8.rotary(48, 1e5, device=DEV)
    for dtype in TYPES:
        y = rnd(n, (nh + 2 * nkv) * hd, seed=3, dtype=dtype).to(DEV)
        norm = (1 + rnd(hd, seed=4) / 4).to(dtype).to(DEV)
        cut = lambda t: (t[:, :nh * hd].view(-1, nh, hd), t[:, nh * hd:(nh + nkv) * hd].view(-1, nkv, hd),  # noqa: E731
                         t[:, (nh + nkv) * hd:].view(-1, nkv, hd))
        first = make_cache([n], nkv, hd)
        want = q8.kv_append(first, *[t.contiguous() for t in cut(y)], i32([n]), rot, starts([n]), n, q_norm=norm, k_norm=norm)
        codes = first.keys.clone(), first.values.clone()

        def again(pages, out, what):
            w = pages.table.cpu()[0].tolist()
            for p, t in enumerate(w):
                m = min(64, n - 64 * p)
                assert torch.equal(pages.keys[t, :, :m, :hd], first.keys[first.table[0, p], :, :m, :hd]), what
                assert torch.equal(pages.values[t, :, :hd, :m], first.values[first.table[0, p], :, :hd, :m]), what
                assert torch.equal(pages.key_scale[t, :, :m], first.key_scale[first.table[0, p], :, :m]), what
            assert torch.equal(out, want), what

        pages = make_cache([n], nkv, hd, seed=2)
        again(pages, q8.kv_append(pages, *cut(y), i32([n]), rot, starts([n]), n, q_norm=norm, k_norm=norm), "slices")
        for pad in (1, 3):  # odd strides and addresses
            wide = torch.zeros(n, y.shape[1] + pad, dtype=dtype, device=DEV)
            wide[:, pad:] = y
            odd = torch.zeros(hd + 1, dtype=dtype, device=DEV)
            odd[1:] = norm
            pages = make_cache([n], nkv, hd, seed=2)
            parts = [t.as_strided((n, h, hd), (wide.stride(0), hd, 1), pad + o) for t, h, o in
                     ((wide, nh, 0), (wide, nkv, nh * hd), (wide, nkv, (nh + nkv) * hd))]
            again(pages, q8.kv_append(pages, *parts, i32([n]), rot, starts([n]), n, q_norm=odd[1:], k_norm=odd[1:]), pad)
        # row by row, in pieces, and in place
        pages = make_cache([n], nkv, hd, seed=2)
        out = torch.empty_like(want)
        at = 0
        for c in (1, 2, 15, 16, 17, 40, 1, 1, 57):
            q, k, v = cut(y[at:at + c])
            at += c
            q8.kv_append(pages, q, k, v, i32([at]), rot, starts([c]), c, q_norm=norm, k_norm=norm, out=out[at - c:at])
        again(pages, out, "pieces")
        own = y.clone()
        q, k, v = cut(own)
        pages = make_cache([n], nkv, hd, seed=2)
        got = q8.kv_append(pages, q, k, v, i32([n]), rot, starts([n]), n, q_norm=norm, k_norm=norm, out=q)
        assert got is q
        again(pages, got, "in place")
        assert torch.equal(own[:, nh * hd:], y[:, nh * hd:])
        assert torch.equal(codes[0], first.keys) and torch.equal(codes[1], first.values)


def test_append_rows_of_no_sequence_bad_pages_and_odd_values():
    lens, nh, nkv, hd = [70, 66], 4, 2, 64
    rot = q8.rotary(hd, device=DEV)
    pages = make_cache(lens, nkv, hd)
    table = pages.table.clone()
    table[0, 1], table[1, 0] = 1000, -5
    pages = pages._replace(table=table)
    before = [t.clone() for t in pages]
    q, k, v = rnd(140, nh, hd, seed=3), rnd(140, nkv, hd, seed=1), rnd(140, nkv, hd, seed=2)
    k[3, 0, 5], v[4, 1, 7], q[6, 2, 40], k[5, 1] = math.inf, math.nan, math.nan, 0
    args = (i32(lens), rot, i32([1, 71, 137]))  # row 0 and the last three are nobody's
    out = q8.kv_append(pages, q.to(DEV), k.to(DEV), v.to(DEV), *args, most_rows=70).cpu()
    assert not out[:1].any() and not out[137:].any()
    assert torch.isnan(out[6, 2, [8, 40]]).all() and int(torch.isnan(out).sum()) == 2
    pos = torch.cat([torch.arange(70), torch.arange(66)])
    want = turned(q[1:137], None, 0, rot.freq.cpu(), False, 1.0, pos)
    assert ((out[1:137].double() - want).abs().nan_to_num() <= 1e-7 * want.abs().nan_to_num() + 1e-11).all()
    p0 = int(table[0, 0])
    assert torch.isnan(pages.key_scale[p0, 0, 2]) and torch.isnan(pages.value_scale[p0, 1, 3]) and pages.key_scale[p0, 1, 4] == 0
    assert not pages.keys[p0, 0, 2].any() and int(torch.isnan(pages.key_scale[p0]).sum()) == 1
    used = {p0, int(table[1, 1])}
    for p in range(len(before[0])):
        if p not in used:
            assert all(same(a[p], b[p]) for a, b in zip(pages[:4], before[:4]))
    into = torch.full((140, nh, hd), 3.0, device=DEV)
    q8.kv_append(pages, q.to(DEV), k.to(DEV), v.to(DEV), *args, most_rows=70, out=into)
    assert (into[0] == 3).all() and (into[137:] == 3).all() and same(into[1:137], out[1:137])
    # more rows than positions: the first ones have no place, but are turned
    fresh = make_cache([4], nkv, hd)
    out = q8.kv_append(fresh, q[20:26].to(DEV), k[20:26].to(DEV), v[20:26].to(DEV), i32([4]), rot, i32([0, 6]), 6).cpu()
    want = turned(q[20:26], None, 0, rot.freq.cpu(), False, 1.0, torch.arange(-2, 4))
    assert ((out.double() - want).abs() <= 1e-7 * want.abs() + 1e-11).all()
    rk, rv = q8.kv_read(fresh, i32([4]), i32([0, 6]), 6, hd)
    assert not rk[:2].any() and ((rv[2:].cpu().double() - values(v[22:26])).abs() <= 1e-6).all()
    # nothing to do, and nothing but what is nobody's
    none = q8.kv_append(fresh, q[:0].to(DEV), k[:0].to(DEV), v[:0].to(DEV), i32([4]), rot, i32([0, 0]))
    assert none.shape == (0, nh, hd)
    assert not q8.kv_append(fresh, q[20:23].to(DEV), k[:3].to(DEV), v[:3].to(DEV), i32([4]), rot, i32([0, 0]), 0).any()
    nobody = fresh._replace(table=fresh.table[:0])
    assert not q8.kv_append(nobody, q[20:23].to(DEV), k[:3].to(DEV), v[:3].to(DEV), i32([]), rot, i32([0])).any()
    # a norm of a head of zeros, and of one whose squares pass f32's range
    w = torch.ones(hd, device=DEV)
    big = torch.stack([torch.zeros(nh, hd), torch.full((nh, hd), 1e30)]).to(DEV)
    out = q8.kv_append(fresh, big, k[:2].to(DEV), v[:2].to(DEV), i32([2]), q8.rotary(0, device=DEV), i32([0, 2]), 2, q_norm=w, eps=0.0)
    assert torch.isnan(out[0]).all() and torch.equal(out[1], torch.ones(nh, hd, device=DEV))


@pytest.mark.parametrize("dtype,hd", [(torch.float32, 64), (torch.float32, 200), (torch.float32, 7), (torch.bfloat16, 128),
                                      (torch.bfloat16, 256)])
def test_append_codes_at_and_beside_halves_of_every_scale(dtype, hd):
    """Without rotation the codes and scales are the cache write's, also of values half-way between codes, of their
    neighbours, and where the scale is near either end of the type's range."""
    powers = (-100, -94, -93, -60, -20, -1, 0, 1, 50, 110, 116, 117, 118, 119, 120)
    g = torch.Generator().manual_seed(hd)
    rows = []
    for e in powers:
        for near in (0, 1, -1):
            codes = torch.randint(-127, 127, (hd,), generator=g).float() + 0.5
            x = codes.to(dtype)
            if near:
                bits = torch.int32 if dtype == torch.float32 else torch.int16
                x = (x.view(bits) + near).view(dtype)  # the next number, or the one before
            x[0] = 127
            rows.append((x.float() * 2.0 ** e).to(dtype))
    x = torch.stack(rows)[:, None].to(DEV)
    n = len(x)
    a, b = make_cache([n], 1, hd, seed=1), make_cache([n], 1, hd, seed=1)
    b.keys.copy_(a.keys)
    b.values.copy_(a.values)
    out = q8.kv_append(a, x, x, x, i32([n]), q8.rotary(0, device=DEV), starts([n]), n)
    q8.kv_write(b, x, x, i32([n]), starts([n]), n)
    assert torch.equal(out, x) and all(same(s, t) for s, t in zip(a, b))


def test_append_of_many_runs_and_of_one_give_the_same_bits():
    """Workgroups take more heads where there are many runs of rows: neither that nor a call's other rows show."""
    nh, nkv, hd, n, seqs = 15, 5, 64, 47, 60
    rot = q8.rotary(hd, 1e4, interleaved=True, device=DEV)
    q, k, v = (rnd(seqs * n, h, hd, seed=i, dtype=torch.bfloat16).to(DEV) for i, h in enumerate((nh, nkv, nkv)))
    lens = [n + 3 * i for i in range(seqs)]
    pages, alone = make_cache(lens, nkv, hd, seed=1), make_cache(lens, nkv, hd, seed=1)
    alone.keys.copy_(pages.keys)
    alone.values.copy_(pages.values)
    out = q8.kv_append(pages, q, k, v, i32(lens), rot, starts([n] * seqs), n)
    for i in range(seqs):
        one = alone._replace(table=alone.table[i:i + 1].contiguous())
        r = slice(i * n, i * n + n)
        assert torch.equal(q8.kv_append(one, q[r], k[r], v[r], i32(lens[i:i + 1]), rot, starts([n]), n), out[r])
    assert all(same(a, b) for a, b in zip(pages, alone))


# ------------------------------------------------------------------ trees

def random_tree(n, seed, back=4):
    g = torch.Generator().manual_seed(seed)
    return [max(-1, i - 1 - int(torch.randint(0, back, (1,), generator=g))) for i in range(n)]


def path_of(parent, j):
    p = []
    while 0 <= j:
        p.append(j)
        j = parent[j] if parent[j] < j else -1
    return p[::-1]


def path_cache(pages, table, n, ctx, path):
    """The pages of one sequence with only this path behind its history, in pages of its own: codes, moved one by one."""
    t = table.tolist()
    blocks = (ctx + len(path) + 63) // 64
    own = q8.Pages(*[x[t[:blocks]].clone() for x in pages[:4]], torch.arange(blocks, dtype=torch.int32, device=DEV)[None])
    for d, i in enumerate(path):
        (pa, a), (pb, b) = divmod(ctx + d, 64), divmod(ctx + i, 64)
        own.keys[pa, :, a], own.key_scale[pa, :, a] = pages.keys[t[pb], :, b], pages.key_scale[t[pb], :, b]
        own.values[pa, :, :, a], own.value_scale[pa, :, a] = pages.values[t[pb], :, :, b], pages.value_scale[t[pb], :, b]
    return own


def check_tree(ctxs, trees, nh, nkv, hd, dtype=torch.float32, hidden=None, seed=0, scale=None, some=None, formula=True):
    """Every node's bits are those of attention over its path alone; and within f32's accuracy of the formula."""
    counts = [len(t) for t in trees]
    lens = [c + n for c, n in zip(ctxs, counts)]
    pages = make_cache(lens, nkv, hd, seed=seed)
    k, v = fill(pages, lens, nkv, hd, seed=seed)
    q = rnd(sum(counts), nh, hd, seed=seed + 7, dtype=dtype).to(DEV)
    hid = None if hidden is None else hidden.to(DEV)
    parent = i32([p for t in trees for p in t])
    out = q8.tree_attention(q, pages, parent, i32(lens), starts(counts), max(counts), max(lens), scale=scale, hidden=hid)
    sc = hd ** -0.5 if scale is None else scale
    at = 0
    for i, (ctx, tree) in enumerate(zip(ctxs, trees)):
        for j in range(len(tree)) if some is None else some:
            path = path_of(tree, j)
            n = ctx + len(path)
            own = path_cache(pages, pages.table[i].cpu(), n, ctx, path)
            h = None
            if hidden is not None:
                h = torch.zeros(1, n, dtype=torch.uint8)
                places = torch.tensor(list(range(ctx)) + [ctx + p for p in path])
                inside = places < hidden.shape[1]
                h[0, inside] = hidden[i, places[inside]].to(torch.uint8)
                h = h.to(DEV)
            one = q8.attention(q[at + j:at + j + 1], own, i32([n]), scale=scale, hidden=h)
            assert same(out[at + j], one[0]), (i, j, ctx, path)
        if formula and tree:
            k0 = sum(lens[:i])
            kd, vd = values(k[k0:k0 + lens[i]]), values(v[k0:k0 + lens[i]])
            off = torch.ones(len(tree), lens[i], dtype=torch.bool)
            off[:, :ctx] = False
            for j in range(len(tree)):
                off[j, [ctx + p for p in path_of(tree, j)]] = False
            for j in range(len(tree)) if some is None else some:
                hj = off[j].clone()
                if hidden is not None:
                    m = min(hidden.shape[1], lens[i])
                    hj[:m] |= hidden[i, :m].bool()
                want, big, mass = ref_attention(q[at + j:at + j + 1].cpu(), kd, vd, [lens[i] - 1], hj, sc)
                got = out[at + j:at + j + 1].cpu().double()
                assert ((got - want).abs() <= tolerance(dtype, lens[i], big, mass, want)).all(), (i, j)
        at += len(tree)
    return q, pages, parent, lens, counts, out


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nh,nkv,hd", [(9, 3, 64), (8, 2, 128), (4, 2, 16), (5, 1, 72), (4, 4, 256), (14, 2, 192), (16, 2, 64)])
def test_tree_rows_have_their_paths_bits(nh, nkv, hd, dtype):
    ctxs = [0, 1, 63, 64, 200, 130, 5, 60]
    trees = [random_tree(n, seed=n) for n in (7, 1, 12, 3, 0, 20, 2, 9)]
    check_tree(ctxs, trees, nh, nkv, hd, dtype=dtype, seed=hd)


@pytest.mark.parametrize("ctx", [0, 33, 64, 127, 300])
def test_trees_of_64_rows(ctx):
    chain, star = list(range(-1, 63)), [-1] * 64
    deep = [-1] + [0] + list(range(1, 31)) + [0] + list(range(32, 63))  # two arms
    some = [0, 1, 2, 31, 32, 33, 40, 62, 63]
    for nh, nkv, hd in ((6, 2, 64), (4, 1, 128)):
        check_tree([ctx] * 4, [chain, star, deep, random_tree(64, 3)], nh, nkv, hd, seed=ctx, some=some, formula=False)


def test_a_chain_is_a_prompt():
    for nh, nkv, hd, ctx, n in ((9, 3, 64, 100, 30), (8, 2, 128, 250, 64), (32, 8, 64, 0, 17), (4, 1, 64, 8150, 60)):
        pages = make_cache([ctx + n, 64], nkv, hd)
        fill(pages, [ctx + n, 64], nkv, hd)
        q = rnd(n + 3, nh, hd, seed=5).to(DEV)
        want = q8.attention(q, pages, i32([ctx + n, 64]), starts([n, 3]), n, ctx + n)
        parent = i32(list(range(-1, n - 1)) + [-1, 0, 1])
        assert torch.equal(q8.tree_attention(q, pages, parent, i32([ctx + n, 64]), starts([n, 3]), n, ctx + n), want)


@pytest.mark.parametrize("seqs", [1, 3, 40])
def test_trees_split_over_workgroups_or_not(seqs):
    """The same trees beside others, enough of them that rows' positions are dealt otherwise."""
    nh, nkv, hd, ctx = 8, 2, 64, 1900
    tree = random_tree(11, 5)
    n = ctx + len(tree)
    pages = make_cache([n], nkv, hd)
    fill(pages, [n], nkv, hd)
    q = rnd(11, nh, hd, seed=3).to(DEV)
    many = pages._replace(table=pages.table.expand(seqs, -1).contiguous())
    out = q8.tree_attention(q.repeat(seqs, 1, 1), many, i32(tree * seqs), i32([n] * seqs), starts([11] * seqs), 11, n)
    for j in (0, 3, 7, 10):
        path = path_of(tree, j)
        own = path_cache(pages, pages.table[0].cpu(), n, ctx, path)
        one = q8.attention(q[j:j + 1], own, i32([ctx + len(path)]))
        for i in (0, seqs // 2, seqs - 1):
            assert torch.equal(out[11 * i + j], one[0])


@pytest.mark.parametrize("nh,nkv,hd", [(64, 8, 64), (64, 8, 40), (32, 8, 128), (48, 8, 72)])
def test_trees_of_many_workgroups_and_of_few_give_the_same_bits(nh, nkv, hd):
    """Where there are many, a wave takes two tiles of rows; the last ones of a sequence are not full."""
    seqs, ctxs = 64 if nh == 64 else 128, (70, 0, 130, 57)
    counts = [(17, 20, 1, 13, 20)[i % 5] for i in range(seqs)]
    trees = [random_tree(c, i) for i, c in enumerate(counts)]
    lens = [ctxs[i % 4] + c for i, c in enumerate(counts)]
    pages = make_cache(lens, nkv, hd, seed=2)
    fill(pages, lens, nkv, hd, seed=2)
    q = rnd(sum(counts), nh, hd, seed=4).to(DEV)
    h = (torch.rand(seqs, 140, generator=torch.Generator().manual_seed(3)) < 0.3).to(DEV)
    for hidden in (None, h):
        out = q8.tree_attention(q, pages, i32(sum(trees, [])), i32(lens), starts(counts), 20, max(lens), hidden=hidden)
        at = 0
        for i, c in enumerate(counts):
            one = pages._replace(table=pages.table[i:i + 1].contiguous())
            alone = q8.tree_attention(q[at:at + c], one, i32(trees[i]), i32(lens[i:i + 1]), starts([c]), c,
                                      hidden=None if hidden is None else hidden[i:i + 1])
            assert torch.equal(out[at:at + c], alone), i
            at += c


def test_trees_across_unit_lengths():
    # units of 128 positions up to 8,192, then 256: nodes on both sides of the border
    for ctx in (8180, 8191, 8128, 8100):
        check_tree([ctx], [random_tree(40, 9, back=3)], 4, 1, 64, seed=1, some=[0, 5, 12, 20, 30, 39], formula=False)
    check_tree([16380], [list(range(-1, 9))], 8, 1, 128, seed=1, some=[0, 3, 4, 9], formula=False)


def test_trees_with_hidden_positions_and_places():
    ctxs, trees = [130, 70, 300, 0, 64], [random_tree(n, n) for n in (30, 1, 7, 64, 5)]
    h = torch.rand(5, 310, generator=torch.Generator().manual_seed(1)) < 0.4
    h[1] = True          # sees nothing
    h[3, :40] = True     # its first rows see nothing
    for hidden in (h, h[:, :150].contiguous(), h.new_zeros(5, 0)):
        out = check_tree(ctxs, trees, 6, 2, 64, hidden=hidden, seed=4)[-1]
        if hidden.shape[1] > 70:
            assert not out[30:31].any()


def test_trees_do_not_see_what_they_must_not():
    """NaN in places of nodes on other paths, in hidden ones and in pages of nobody changes nothing."""
    tree = [-1, 0, 0, 1, 2, 3, -1]
    for ctx in (50, 60, 64):
        lens = [ctx + 7]
        pages = make_cache(lens, 2, 64)
        fill(pages, lens, 2, 64)
        q = rnd(7, 6, 64, seed=9).to(DEV)
        args = (i32(tree), i32(lens), starts([7]), 7)
        want = q8.tree_attention(q, pages, *args)
        bad = q8.Pages(*[t.clone() for t in pages])
        page, place = divmod(ctx + 3, 64)
        p = int(pages.table[0, page])
        bad.key_scale[p, :, place] = math.nan
        bad.value_scale[p, :, place] = math.inf
        bad.keys[p, :, place], bad.values[p, :, :, place] = 127, -128
        out = q8.tree_attention(q, bad, *args)
        for j in range(7):
            if 3 in path_of(tree, j):
                assert torch.isnan(out[j]).all()
            else:
                assert torch.equal(out[j], want[j])
        h = torch.zeros(1, ctx + 7, dtype=torch.uint8, device=DEV)
        h[0, ctx + 3] = 1
        assert torch.equal(q8.tree_attention(q, bad, *args, hidden=h), q8.tree_attention(q, pages, *args, hidden=h))


def test_trees_of_bad_parents_lengths_and_pages():
    lens, nh, nkv, hd = [100, 9], 4, 2, 64
    pages = make_cache(lens, nkv, hd)
    fill(pages, lens, nkv, hd)
    q = rnd(12, nh, hd, seed=3).to(DEV)
    args = (i32(lens), starts([7, 5]), 7, 100)
    good = q8.tree_attention(q, pages, i32([-1, 0, -1, -1, 3, -1, 5, -1, -1, 1, -1, 3]), *args)
    # no earlier row: itself, a later one, none of the call's
    out = q8.tree_attention(q, pages, i32([0, 0, 2, 5, 3, 2 ** 31 - 1, 5, -7, -2 ** 31, 1, 64, 3]), *args)
    assert torch.equal(out, good)
    # a sequence of fewer positions than rows has no history that its rows could follow
    out = q8.tree_attention(q, pages, i32([-1, 0, 1, 2, 3, 4, 5, -1, 0, 1, 2, 3]), i32([100, 4]), starts([7, 5]), 7, 100)
    assert not out[7:].any() and out[:7].any()
    assert not q8.tree_attention(q, pages, i32([-1] * 12), i32([-2 ** 31, 0]), starts([7, 5]), 7, 100).any()
    # rows of nobody
    into = torch.full((12, nh, hd), 3.0, device=DEV)
    got = q8.tree_attention(q, pages, i32([-1] * 12), i32(lens), i32([1, 8, 11]), 7, 100, out=into)
    assert got is into and (into[0] == 3).all() and (into[11] == 3).all() and not (into[1:11] == 3).any()
    clear = q8.tree_attention(q, pages, i32([-1] * 12), i32(lens), i32([1, 8, 11]), 7, 100)
    assert not clear[0].any() and not clear[11].any() and torch.equal(clear[1:11], into[1:11])
    own = q.clone()
    assert torch.equal(q8.tree_attention(own, pages, i32([-1] * 12), i32(lens), i32([1, 8, 11]), 7, 100, out=own)[1:11], into[1:11])
    assert q8.tree_attention(q[:0], pages, i32([]), i32(lens), i32([0, 0, 0])).shape == (0, nh, hd)
    # pages that are not there hide what they would hold: history, or drafted places
    ctx, tree = 120, random_tree(16, 2)
    pages = make_cache([136], nkv, hd)
    fill(pages, [136], nkv, hd)
    q = rnd(16, nh, hd, seed=4).to(DEV)
    for gone in (0, 1, 2):
        table = pages.table.clone()
        table[0, gone] = -1
        h = torch.zeros(1, 136, dtype=torch.uint8, device=DEV)
        h[0, 64 * gone:64 * gone + 64] = 1
        a = q8.tree_attention(q, pages._replace(table=table), i32(tree), i32([136]), starts([16]), 16)
        assert torch.equal(a, q8.tree_attention(q, pages, i32(tree), i32([136]), starts([16]), 16, hidden=h)), gone
    # most_len: positions behind it are not attended to
    short = q8.tree_attention(q, pages, i32([-1] * 16), i32([136]), starts([16]), 16, most_len=64)
    h = torch.zeros(1, 136, dtype=torch.uint8, device=DEV)
    h[0, 64:] = 1
    assert torch.allclose(short, q8.tree_attention(q, pages, i32([-1] * 16), i32([136]), starts([16]), 16, hidden=h), atol=1e-6)


# ------------------------------------------------------------------ keep

@pytest.mark.parametrize("heads,hd", [(1, 1), (3, 64), (2, 40), (8, 128), (1, 256)])
def test_keep(heads, hd):
    lens, counts = [70, 64, 130, 5, 200, 90], [7, 64, 64, 5, 1, 0]
    pages = make_cache(lens, heads, hd, seed=hd)
    fill(pages, lens, heads, hd, seed=hd)
    g = torch.Generator().manual_seed(hd)
    keep, kept = [], []
    for i, n in enumerate(counts):
        if i == 2:
            which = list(range(1, 64, 2)) + [0, 0, 63]  # out of order, and one twice
        else:
            which = sorted(torch.randperm(n, generator=g)[:n * 2 // 3].tolist())
        kept.append(len(which))
        keep += which + [-1] * (n - len(which))
    old = q8.kv_read(pages, i32(lens), starts(counts), sum(counts), hd)
    before = [t.clone() for t in pages]
    got = q8.kv_keep(pages, i32(lens), starts(counts), i32(keep), i32(kept), 64)
    want = [n - c + m for n, c, m in zip(lens, counts, kept)]
    assert got.tolist() == want and got.dtype == torch.int32
    new = q8.kv_read(pages, got, starts(kept), sum(kept), hd)
    rows = [sum(counts[:i]) + keep[sum(counts[:i]) + t] for i, m in enumerate(kept) for t in range(m)]
    for a, b in zip(new, old):
        assert torch.equal(a, b[rows])
    # no other place has changed
    touched = torch.zeros(before[0].shape[0], q8.PAGE, dtype=torch.bool, device=DEV)
    table = pages.table.cpu()
    for i, m in enumerate(kept):
        for t in range(m):
            p = lens[i] - counts[i] + t
            touched[table[i, p // 64], p % 64] = True
    t = touched[:, None].expand(-1, heads, -1)
    assert torch.equal(pages.keys[~t], before[0][~t]) and torch.equal(pages.values.transpose(2, 3)[~t], before[1].transpose(2, 3)[~t])
    assert same(pages.key_scale[~t], before[2][~t]) and same(pages.value_scale[~t], before[3][~t])


def test_keep_of_bad_entries_lengths_and_pages():
    lens = [10, 70]
    pages = make_cache(lens, 2, 64)
    fill(pages, lens, 2, 64)
    before = [t.clone() for t in pages]
    # entries that are no row leave their place; kept past the rows, and below 0
    got = q8.kv_keep(pages, i32(lens), starts([4, 3]), i32([-1, 9, 3, 2 ** 31 - 1, 1, 1, 1]), i32([100, -5]), 4)
    assert got.tolist() == [10, 67]
    p = int(pages.table[0, 0])
    want = before[0].clone()
    want[p, :, 8] = before[0][p, :, 9]
    assert torch.equal(pages.keys, want)
    # places before 0 and pages that are not there
    table = pages.table.clone()
    table[1, 1] = -1
    before = [t.clone() for t in pages]
    got = q8.kv_keep(pages._replace(table=table), i32([2, 66]), starts([4, 4]), i32([1, 2, 3, 3, 3, 2, 1, 0]), i32([2, 4]), 4)
    assert got.tolist() == [0, 66]
    assert all(same(a, b) for a, b in zip(pages, before))
    assert q8.kv_keep(pages, i32(lens), i32([0, 0, 0]), i32([]), i32([1, 1])).tolist() == lens
    assert q8.kv_keep(pages, i32(lens), None, i32([0, 0]), i32([1, 0])).tolist() == [10, 69]
    assert all(same(a, b) for a, b in zip(pages, before))


# ------------------------------------------------------------------ log probabilities

def ref_scores(x, target, top, scale):
    x = x.double()
    y = x * scale
    lp = torch.log_softmax(y, -1)
    p = lp.exp()
    d = torch.where(p > 0, y - y.amax(-1, keepdim=True), torch.zeros_like(y))
    ent = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(-1)
    order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top]
    has = (target >= 0) & (target < x.shape[1])
    t = torch.where(has, target, torch.zeros_like(target)).long()[:, None]
    log_p = torch.where(has, lp.gather(1, t)[:, 0], torch.tensor(math.nan, dtype=torch.float64))
    rank = torch.where(has, (x > x.gather(1, t)).sum(1), torch.tensor(-1))
    return log_p, ent, rank, order, lp.gather(1, order), (p * d.abs()).sum(-1), (p * d * d).sum(-1)


def check_scores(x, target, top, scale=1.0, x_gpu=None):
    got = q8.log_probs(x.to(DEV) if x_gpu is None else x_gpu, None if target is None else target.to(DEV), top, scale)
    t = torch.full((len(x),), -1) if target is None else target
    log_p, ent, rank, order, top_lp, mean, square = ref_scores(x, t, top, scale)
    assert [a.dtype for a in got] == [torch.float32] * 2 + [torch.int32] * 2 + [torch.float32]
    assert torch.equal(got.rank.cpu(), rank.int()) and torch.equal(got.top_index.cpu(), order.int())
    # A term e = exp(t), t = scale d, d = x - max: scale * log2(e) (twice) and the fused product, or d and a product:
    # half a step each, 4 u |t| of e; the exponential a step, 2 u. The sum: 16 terms a lane, 6 steps a wave, the
    # power it is taken back by: under 37 u. So the sum's logarithm is off by u (4 mean |t| + 39); waves join in
    # 64 bits. The moment's terms have one product more and t itself, its sum as many roundings.
    u = 2.0 ** -24
    off = u * (4 * mean + 39)
    assert (got.entropy.cpu().double() - ent).abs().le(off * (1 + mean) + u * (4 * square + 42 * mean) + 1.01 * u * ent).all()
    for a, want in ((got.log_p, log_p), (got.top_log_p, top_lp)):
        a, o = a.cpu().double(), off if want.dim() == 1 else off[:, None]
        assert torch.equal(torch.isnan(a), torch.isnan(want)) and torch.equal(torch.isinf(a), torch.isinf(want.float()))
        fin = torch.isfinite(want.float())
        assert ((a - want).abs() <= o + 1.01 * u * want.abs())[fin].all()
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n,top", [(1, 1, 1), (3, 2, 2), (2, 31, 5), (5, 300, 20), (2, 1000, 32), (3, 16383, 1), (3, 16384, 8),
                                        (3, 16385, 32), (2, 49152, 5), (4, 50001, 0), (2, 128256, 20)])
def test_log_probs(rows, n, top, dtype):
    x = (rnd(rows, n, seed=n) * (1 + torch.arange(rows)[:, None])).to(dtype)
    target = torch.randint(0, n, (rows,), generator=torch.Generator().manual_seed(n), dtype=torch.int32)
    target[0] = int(x[0].float().argmax())
    check_scores(x, target, top)
    check_scores(x, target, top, scale=0.3)
    check_scores(x, None, top, scale=2.5)
    banned = x.clone()
    banned[torch.rand(x.shape, generator=torch.Generator().manual_seed(1)) < 0.7] = -math.inf
    banned[:, n // 2] = x[:, n // 2]
    check_scores(banned, target, top)


def test_log_probs_of_the_largest_rows():
    x = rnd(2, 1 << 20, seed=1) * 3
    check_scores(x, torch.tensor([1, (1 << 20) - 1], dtype=torch.int32), 32)
    x = torch.sort(x, -1, descending=True).values  # all the best in one place
    check_scores(x, torch.tensor([7, 500000], dtype=torch.int32), 32)


@pytest.mark.parametrize("n", [5, 700, 20000, 49152])
def test_log_probs_of_equal_logits(n):
    x = torch.zeros(4, n)
    x[1] = -0.0
    x[1, ::3] = 0.0
    x[2] = torch.round(rnd(n, seed=1) * 2)  # few values, each many times
    x[3] = -math.inf
    x[3, n // 3], x[3, n - 1] = 1.0, 1.0
    target = torch.tensor([n - 1, 1, 3, 0], dtype=torch.int32)
    for top in (1, min(n, 32)):
        got = check_scores(x, target, top)
        assert got.rank.tolist()[:2] == [0, 0] and got.rank.tolist()[3] == 2
        assert got.top_index[0].tolist() == list(range(top))


@pytest.mark.parametrize("dtype", TYPES)
def test_log_probs_of_rows_whose_best_lie_together(dtype):
    """More logits over any bound from groups' maxima than are held at once: in order, in blocks of columns, and equal."""
    n = 49152
    x = rnd(6, n, seed=5)
    x[0] = torch.sort(x[0]).values
    x[1] = torch.sort(x[1], descending=True).values
    c = torch.arange(n)
    for r, w in ((2, 32), (3, 64)):  # 31 of every 64 runs of 32, or 64, columns are far over the rest
        x[r] = x[r] / 8 + torch.where(c // w % 64 < 31, 20.0, 0.0)
    x[4] = torch.where(c // 32 % 64 < 31, torch.round(x[4]) + 8, x[4] - 20)
    x[5] = torch.where(c % 3 == 0, 2.0, torch.where(c == 5, 3.0, -1.0))
    for top in (1, 31, 32):
        check_scores(x.to(dtype), torch.tensor([0, 1, 2, 3, 4, 5], dtype=torch.int32), top)


def test_log_probs_of_logits_at_both_ends_of_the_range():
    for n in (3 * 8192, 9000):
        x = torch.full((4, n), -3e38)
        x[0, 5] = 3e38
        x[1, :n // 2] = 3e38
        x[2] = rnd(n, seed=1) * 1e38
        x[3, ::2], x[3, 1::2] = -math.inf, 1e38
        assert (x[2] == math.inf).any()  # 3.4 standard deviations, and so no distribution
        got = q8.log_probs(x[2:3].to(DEV), torch.tensor([3], dtype=torch.int32).to(DEV), 4)
        assert torch.isnan(got.log_p[0]) and torch.isnan(got.entropy[0]) and got.rank[0] == -1 and (got.top_index[0] == -1).all()
        x[2] = rnd(n, seed=1) * 5e37
        got = check_scores(x, torch.tensor([5, 0, 3, 1], dtype=torch.int32), 4)
        assert got.entropy[0] == 0 and abs(float(got.entropy[1]) - math.log(n // 2)) < 1e-5 and got.log_p[0] == 0
        for scale in (1e-30, 1e30):
            check_scores(rnd(3, n, seed=2), torch.tensor([1, 2, 3], dtype=torch.int32), 4, scale=scale)
        check_scores(x[2:3] / 8, torch.tensor([1], dtype=torch.int32), 4, scale=1e-30)


def test_log_probs_of_rows_without_a_distribution():
    for n in (40, 33000):
        x = rnd(7, n, seed=2)
        x[1, n - 1] = math.nan
        x[2, 3] = math.inf
        x[3] = -math.inf
        x[4] = math.nan
        x[5, :n - 1] = -math.inf
        target = torch.tensor([0, 0, 0, 0, 0, n - 1, n], dtype=torch.int32)
        got = q8.log_probs(x.to(DEV), target.to(DEV), 3)
        for r in (1, 2, 3, 4):
            assert all(torch.isnan(t[r]).all() for t in (got.log_p, got.entropy, got.top_log_p))
            assert got.rank[r] == -1 and (got.top_index[r] == -1).all()
        check_scores(x[:1], target[:1], 3)
        assert got.log_p[5] == 0 and got.entropy[5] == 0 and got.rank[5] == 0
        assert got.top_index[5].tolist() == [n - 1, 0, 1] and torch.isinf(got.top_log_p[5, 1:]).all()
        assert torch.isnan(got.log_p[6]) and got.rank[6] == -1 and torch.isfinite(got.entropy[6])
        check_scores(x[6:], target[6:], 3)
    # far out in f32's range
    x = torch.tensor([[3e38, -3e38, 2.9e38], [1e-40, 0.0, -1e-40], [-3e38, -3e38, -3.1e38]])
    got = check_scores(x, torch.tensor([2, 1, 0], dtype=torch.int32), 3)
    assert got.entropy[0] == 0 and abs(float(got.entropy[1]) - math.log(3)) < 1e-6
    assert q8.log_probs(x[:0].to(DEV), None, 2).top_index.shape == (0, 2)


@pytest.mark.parametrize("dtype", TYPES)
def test_log_probs_strides_and_calls_give_the_same_bits(dtype):
    n = 33001
    x = (rnd(40, n, seed=3) * 2).to(dtype).to(DEV)
    target = torch.arange(40, dtype=torch.int32, device=DEV) * 800
    want = q8.log_probs(x, target, 7)
    for pad in (1, 7, 8):
        wide = torch.zeros(40, n + pad, dtype=dtype, device=DEV)
        wide[:, pad:] = x
        assert all(torch.equal(a, b) for a, b in zip(q8.log_probs(wide[:, pad:], target, 7), want))
    for a, b in ((0, 1), (5, 8), (39, 40)):
        assert all(torch.equal(s, t[a:b]) for s, t in zip(q8.log_probs(x[a:b], target[a:b], 7), want))
    again = q8.log_probs(x[::2], target[::2].contiguous(), 3)
    assert torch.equal(again.log_p, want.log_p[::2]) and torch.equal(again.top_index, want.top_index[::2, :3])


# ------------------------------------------------------------------ together

class Model:
    """A model of one layer on the 8-bit operators, enough to decode with."""

    def __init__(self, vocab=300, h=64, nh=4, nkv=2, hd=32):
        self.h, self.nh, self.nkv, self.hd, self.vocab = h, nh, nkv, hd, vocab
        g = lambda *s, seed: rnd(*s, seed=seed).to(DEV)  # noqa: E731
        self.embed = g(vocab, h, seed=1)
        self.norm, self.qn, self.kn = torch.ones(h, device=DEV), 1 + g(hd, seed=2) / 4, 1 + g(hd, seed=3) / 4
        self.qkv, self.o, self.head = (q8.quantize(g(m, k, seed=4 + m) * k ** -0.5)
                                       for m, k in (((nh + 2 * nkv) * hd, h), (h, nh * hd), (vocab, h)))
        self.rot = q8.rotary(hd, 1e4, interleaved=True, device=DEV)

    def rows(self, tokens, pages, kv_len, row_start, most, position=None, parent=None):
        x = self.embed[tokens]
        _, c, s = q8.rms_norm(x, self.norm, 1e-5)
        y = q8.linear(c, s, *self.qkv).view(len(x), -1, self.hd)
        a, b = self.nh, self.nh + self.nkv
        q = q8.kv_append(pages, y[:, :a], y[:, a:b], y[:, b:], kv_len, self.rot, row_start, most, position=position,
                         q_norm=self.qn, k_norm=self.kn, out=y[:, :a])
        if parent is None:
            z = q8.attention(q, pages, kv_len, row_start, most)
        else:
            z = q8.tree_attention(q, pages, parent, kv_len, row_start, most)
        z, c, s = q8.rms_norm(q8.linear(*q8.quantize(z.reshape(len(x), -1)), *self.o), self.norm, 1e-5, residual=x)
        return q8.linear(c, s, *self.head)


def test_drafted_and_plain_decoding_are_the_same():
    """Sessions that decode token by token, and sessions that verify trees of drafts and keep what was right: the
    same tokens, log probabilities and caches, bit for bit."""
    m, seqs, steps = Model(), 3, 60
    g = torch.Generator().manual_seed(5)
    prompts = [torch.randint(0, m.vocab, (n,), generator=g).tolist() for n in (5, 64, 61)]
    lens = [len(p) for p in prompts]

    def fresh():
        return q8.new_pages(3 * seqs, m.nkv, m.hd, torch.arange(3 * seqs, dtype=torch.int32, device=DEV).view(seqs, 3))

    def prompt(pages):
        x = m.rows(torch.tensor(sum(prompts, [])).to(DEV), pages, i32(lens), starts(lens), max(lens))
        last = (starts(lens)[1:] - 1).long()
        return q8.log_probs(x[last].contiguous(), None, 1).top_index[:, 0].tolist()

    pages = fresh()
    token = prompt(pages)
    plain, scores = [[t] for t in token], [[] for _ in range(seqs)]
    for s in range(steps):
        x = m.rows(torch.tensor([p[-1] for p in plain], device=DEV), pages, i32([n + s + 1 for n in lens]), None, 1)
        best = q8.log_probs(x, None, 3)
        for i in range(seqs):
            plain[i].append(int(best.top_index[i, 0]))
            scores[i].append(best.top_log_p[i].tolist())
    plain_pages = pages

    pages = fresh()
    token = prompt(pages)
    out, got = [[t] for t in token], [[] for _ in range(seqs)]
    length = list(lens)
    while min(len(o) for o in out) < steps + 1:
        tokens, parents, depths, counts = [], [], [], []
        for i in range(seqs):
            n = int(torch.randint(2, 12, (1,), generator=g))
            parent = [-1] + [max(0, j - int(torch.randint(1, 4, (1,), generator=g))) for j in range(1, n)]
            depth = [0] * n
            for j in range(1, n):
                depth[j] = depth[parent[j]] + 1
            tree = [out[i][-1]]
            for j in range(1, n):  # some drafts are right, others wrong
                at = len(out[i]) - 1 + depth[j]
                right = at < len(plain[i]) and bool(torch.rand(1, generator=g) < 0.8)
                tree.append(plain[i][at] if right else int(torch.randint(0, m.vocab, (1,), generator=g)))
            tokens += tree
            parents += parent
            depths += [length[i] + d for d in depth]
            counts.append(n)
        total = [length[i] + counts[i] for i in range(seqs)]
        x = m.rows(torch.tensor(tokens, device=DEV), pages, i32(total), starts(counts), max(counts), position=i32(depths),
                   parent=i32(parents))
        best = q8.log_probs(x, None, 3)
        keep, kept = [], []
        for i in range(seqs):
            r0 = sum(counts[:i])
            path = [0]
            while True:
                at = r0 + path[-1]
                out[i].append(int(best.top_index[at, 0]))
                got[i].append(best.top_log_p[at].tolist())
                child = [j for j in range(path[-1] + 1, counts[i]) if parents[r0 + j] == path[-1] and tokens[r0 + j] == out[i][-1]]
                if not child:
                    break
                path.append(child[0])
            kept.append(len(path))
            keep += path + [-1] * (counts[i] - len(path))
        length = q8.kv_keep(pages, i32(total), starts(counts), i32(keep), i32(kept), max(counts)).tolist()
    for i in range(seqs):
        assert out[i][:steps + 1] == plain[i] and got[i][:steps] == scores[i]
    both = [n + steps for n in lens]
    for a, b in zip(q8.kv_read(pages, i32(both), starts(both), sum(both), m.hd),
                    q8.kv_read(plain_pages, i32(both), starts(both), sum(both), m.hd)):
        assert torch.equal(a, b)


def test_a_verifying_step_in_a_graph_and_on_streams():
    m = Model()
    n, counts, parent = [40, 75], [6, 9], random_tree(6, 1) + random_tree(9, 2)
    table = torch.arange(6, dtype=torch.int32, device=DEV).view(2, 3)
    tokens = torch.randint(0, m.vocab, (15,), generator=torch.Generator().manual_seed(2)).to(DEV)
    kv_len, start = i32(n), starts(counts)
    position = i32([a - c + len(path_of(parent[o:o + c], j)) - 1 for a, c, o in zip(n, counts, (0, 6)) for j in range(c)])
    keep, kept = i32([0, 2, 3, -1, -1, -1, 1, 4, -1, -1, -1, -1, -1, -1, -1]), i32([3, 2])
    history = q8.new_pages(6, m.nkv, m.hd, table)
    hk = rnd(100, m.nkv, m.hd, seed=8).to(DEV)
    q8.kv_write(history, hk, hk, i32([34, 66]), starts([34, 66]), 66)

    def step(pages):
        x = m.rows(tokens, pages, kv_len, start, 9, position=position, parent=i32_parent)
        return tuple(q8.log_probs(x, target, 4)) + (q8.kv_keep(pages, kv_len, start, keep, kept, 9),)

    i32_parent, target = i32(parent), torch.zeros(15, dtype=torch.int32, device=DEV)

    def eager():
        pages = q8.Pages(*[t.clone() for t in history[:4]], table)
        return step(pages), pages

    want, want_pages = eager()
    pages = q8.Pages(*[t.clone() for t in history[:4]], table)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(pages)
    torch.cuda.current_stream().wait_stream(side)
    assert all(same(a, b) for a, b in zip(got, want)) and all(same(a, b) for a, b in zip(pages, want_pages))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(pages)
    for seed in range(4):
        tokens.copy_(torch.randint(0, m.vocab, (15,), generator=torch.Generator().manual_seed(seed)))
        target.copy_(tokens)
        for a, b in zip(pages[:4], history[:4]):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        want, want_pages = eager()
        assert all(same(a, b) for a, b in zip(got, want)) and all(same(a, b) for a, b in zip(pages, want_pages))
        assert i8(1, 1).numel() == 1 and torch.randn(100, device=DEV).sum().item() is not None  # the program's own work between


def test_calls_without_row_start_and_defaults():
    """One row of each sequence without row_start; most_rows and most_len as the call can know them."""
    lens, nh, nkv, hd = [70, 1, 64, 200], 6, 2, 64
    pages, other = make_cache(lens, nkv, hd), make_cache(lens, nkv, hd)
    fill(pages, lens, nkv, hd)
    fill(other, lens, nkv, hd)
    q, k, v = (rnd(4, h, hd, seed=i).to(DEV) for i, h in enumerate((nh, nkv, nkv)))
    rot = q8.rotary(hd, device=DEV)
    a = q8.kv_append(pages, q, k, v, i32(lens), rot)
    b = q8.kv_append(other, q, k, v, i32(lens), rot, starts([1] * 4))
    assert torch.equal(a, b)
    assert torch.equal(*(torch.cat([t.float().flatten() for t in q8.kv_read(p, i32(lens), starts(lens), sum(lens), hd)])
                         for p in (pages, other)))
    root = i32([-1] * 4)
    want = q8.attention(a, pages, i32(lens))
    assert torch.equal(q8.tree_attention(a, pages, root, i32(lens)), want)
    assert torch.equal(q8.tree_attention(a, pages, root, i32(lens), starts([1] * 4)), want)
    assert q8.kv_keep(pages, i32(lens), None, i32([0] * 4), i32([1, 1, 0, 1])).tolist() == [70, 1, 63, 200]
    # 140 rows of three sequences, at most 64 each
    counts = [64, 12, 64]
    big = make_cache([64, 90, 300], nkv, hd)
    fill(big, [64, 90, 300], nkv, hd)
    q = rnd(140, nh, hd, seed=5).to(DEV)
    tree = i32(sum((random_tree(n, n) for n in counts), []))
    args = (q, big, tree, i32([64, 90, 300]), starts(counts))
    assert torch.equal(q8.tree_attention(*args), q8.tree_attention(*args, 64, 300))
    with pytest.raises(ValueError, match="at most 64"):
        q8.tree_attention(*args, 65)
    with pytest.raises(ValueError, match="at most 64"):
        q8.kv_keep(big, i32([64, 90, 300]), starts(counts), tree, i32([0, 0, 0]), 65)


def test_what_calls_write_has_a_new_version():
    lens = [70]
    pages = make_cache(lens, 2, 64)
    fill(pages, lens, 2, 64)
    q, k = rnd(4, 4, 64, seed=1).to(DEV), rnd(4, 2, 64, seed=2).to(DEV)
    out, rot, before = torch.empty_like(q), q8.rotary(64, device=DEV), [t._version for t in pages]
    q8.kv_append(pages, q, k, k, i32(lens), rot, starts([4]), out=out)
    assert out._version == 1 and [t._version for t in pages] == [n + 1 for n in before[:4]] + before[4:]
    q8.tree_attention(q, pages, i32([-1, 0, 0, 1]), i32(lens), starts([4]), out=out)
    assert out._version == 2 and q._version == k._version == 0
    q8.kv_keep(pages, i32(lens), starts([4]), i32([0, 2, 2, 2]), i32([2]))
    assert [t._version for t in pages] == [n + 2 for n in before[:4]] + before[4:]


def test_two_calls_at_once_have_workspaces_of_their_own():
    """On two streams, each of them in turn, and in two graphs that are replayed together."""
    nh, nkv, hd, lens, counts = 8, 2, 64, [1900, 800], [9, 20]
    pages = make_cache(lens, nkv, hd)
    fill(pages, lens, nkv, hd)
    tree = i32(random_tree(9, 1) + random_tree(20, 2))
    qs = [rnd(29, nh, hd, seed=i).to(DEV) for i in range(2)]
    xs = [rnd(29, 50000, seed=i).to(DEV) for i in range(2)]
    target, kv_len, start = i32(list(range(29))), i32(lens), starts(counts)

    def work(i):
        return (q8.tree_attention(qs[i], pages, tree, kv_len, start, 20, 1900),) + tuple(q8.log_probs(xs[i], target, 20))

    want = [work(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        got = []
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got.append(work(i))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))
    graphs, got = [], []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            got.append(work(i))
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g, w in zip(got, want) for a, b in zip(g, w))
        assert torch.randn(100, device=DEV).sum().item() is not None
