"""The operators that verify drafted tokens over the 8-bit cache, as a user's program calls them, for
timing and comparison.

A program that drafts a tree of tokens and verifies it in one step appends the
drafted rows to the cache with their rotary positions, attends from every node
to the history and to its own ancestors, scores the nodes' tokens, and moves the
path that it accepts together. ``kind`` says which operator a pass runs:

* ``append``  queries and keys normed for each head (``norm``) and rotated, queries returned, keys and values
              quantised into the pages and read back: ``rotated`` values of a head, in pairs side by side
              (``interleaved``) or half apart, at frequencies of ``theta`` slowed down by ``scale`` where they are
              long beside ``original``; rows at the end of their sequences, or nodes of trees (``tree``);
* ``tree``    attention of ``rows`` drafted nodes of each sequence over its history and their ancestors,
              ``hidden`` of 1000 positions hidden;
* ``score``   log probabilities of given tokens among ``n`` logits, their entropy, the tokens' ranks and the
              ``top`` likeliest tokens, ``banned`` of 1000 logits -inf, rows ``pad`` values further apart than they are long;
* ``keep``    ``kept`` of ``rows`` drafted rows of each sequence moved together behind its history and read back.

Rows are held in 8 bits and caches in pages as ``perf/operators.py`` says: n
codes in [-127, 127] and one float32 scale = max / 127, positions 64 j .. 64 j +
63 of sequence i in page ``table[i, j]``, values transposed in their page.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda:0"
PAGE = 64
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SIZE = {"float32": 4, "bfloat16": 2, "float16": 2}
# query heads, cache heads, head size, base of the rotary frequencies, tokens of the shapes the framework runs
SHAPES = {"smollm2-135m": (9, 3, 64, 1e5, 49152), "smollm2-360m": (15, 5, 64, 1e5, 49152),
          "llama-3.2-1b": (32, 8, 64, 5e5, 128256), "llama-3-8b": (32, 8, 128, 5e5, 128256)}


def listed():
    return [
        # One token of one session on the smallest shape: latency counts.
        _append("append-step-135m", **_heads("smollm2-135m"), seqs=1, ctx=203, rows=1, type="float32"),
        # 64 sessions in lockstep far into long contexts, frequencies scaled for them.
        _append("append-lockstep-1b", **_heads("llama-3.2-1b"), seqs=64, ctx=30000, rows=1, type="float32", scale=8.0,
                original=8192),
        # A prompt's rows on the largest shape.
        _append("append-prompt-8b", **_heads("llama-3-8b"), seqs=1, ctx=301, rows=2000, type="bfloat16"),
        # Drafted trees, with norms for each head and pairs side by side in part of the head.
        _append("append-tree-normed", heads=24, kv_heads=4, head_dim=96, theta=1e4, seqs=11, ctx=700, rows=33, type="float16",
                rotated=48, interleaved=True, norm=True, tree=True),
        # A few drafted tokens of one session.
        _tree("tree-step-135m", **_heads("smollm2-135m"), seqs=1, ctx=203, rows=7, type="float32"),
        # 32 sessions in lockstep, a small tree each, some positions hidden.
        _tree("tree-lockstep-1b", **_heads("llama-3.2-1b"), seqs=32, ctx=384, rows=12, type="float32", hidden=20),
        # A few long sessions.
        _tree("tree-long-8b", **_heads("llama-3-8b"), seqs=7, ctx=6000, rows=25, type="bfloat16"),
        # The next token of one session.
        _case("score", "score-step-135m", rows=1, n=49152, top=5, banned=0, pad=0, type="float32"),
        # A tree's nodes, of logits that lie in wider rows.
        _case("score", "score-tree-1b", rows=61, n=128256, top=8, banned=5, pad=13, type="float32"),
        # A whole prompt scored.
        _case("score", "score-prompt-8b", rows=2047, n=128256, top=20, banned=0, pad=0, type="bfloat16"),
        # The accepted path of one session.
        _case("keep", "keep-step-135m", **_heads("smollm2-135m"), seqs=1, ctx=203, rows=7, kept=3),
        # The accepted paths of 64 sessions' larger trees.
        _case("keep", "keep-lockstep-8b", **_heads("llama-3-8b"), seqs=64, ctx=1000, rows=47, kept=9),
    ]


def _heads(shape):
    nh, nkv, hd, theta, _ = SHAPES[shape]
    return {"heads": nh, "kv_heads": nkv, "head_dim": hd, "theta": theta}


def _case(kind, name=None, **kw):
    c = {"kind": kind, **kw}
    if name:
        c["name"] = name
    return c


def _append(name=None, **kw):
    return _case("append", name, **{"rotated": kw["head_dim"], "interleaved": False, "norm": False, "scale": 1.0,
                                    "original": 0, "tree": False, **kw})


def _tree(name=None, **kw):
    return _case("tree", name, **{"hidden": 0, **kw})


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "tree", "tree", "tree", "score", "score", "keep"])
    type_ = rng.choice(["float32", "float32", "bfloat16", "float16"])
    if kind == "score":
        n = rng.choice([rng.choice(list(SHAPES.values()))[4], _log_int(rng, 300, 130000)])
        rows = min(rng.choice([rng.randint(1, 64), _log_int(rng, 1, 2047)]), 2047 * 128256 // (2 * n))
        if type_ == "float32":
            rows = (rows + 1) // 2
        return _case(kind, rows=rows, n=n, top=rng.choice([0, 1, 5, 8, 20, 32]), banned=rng.choice([0, 0, 5, 900]),
                     pad=rng.choice([0, 0, 7, 64]), type=type_)
    heads = _heads(rng.choice(list(SHAPES)))
    if rng.random() < 0.35:  # any other layout
        nkv = rng.choice([1, 2, 4, 6])
        heads = {"heads": nkv * rng.choice([1, 2, 5, 7, 8]), "kv_heads": nkv,
                 "head_dim": rng.choice([16, 40, 64, 80, 96, 128, 200, 256]), "theta": rng.choice([1e4, 1e6])}
    if kind == "append":
        hd, drafted = heads["head_dim"], rng.random() < 0.4
        if drafted or rng.random() < 0.4:  # trees, or a token each, of some sessions
            seqs = _log_int(rng, 1, 64)
            rows = rng.randint(2, 64) if drafted else 1
            rows = max(1, min(rows, 16000 * 128 // (seqs * heads["heads"] * hd)))
        else:
            seqs = rng.choice([1, 1, 3])
            rows = _log_int(rng, 2, max(3, min(2000, 60000 * 128 // (heads["heads"] * hd)) // seqs))
        scale = rng.choice([1.0, 1.0, 4.0, 8.0])
        return _append(**heads, seqs=seqs, ctx=_log_int(rng, 1, 40000 // seqs + 50), rows=rows, type=type_,
                       rotated=rng.choice([hd, hd, hd // 2, hd // 4]), interleaved=rng.random() < 0.4, norm=rng.random() < 0.4,
                       scale=scale, original=rng.choice([0, 8192]) if scale > 1 else 0, tree=drafted)
    seqs = _log_int(rng, 1, 64)
    per = heads["kv_heads"] * heads["head_dim"]
    if kind == "keep":
        rows = rng.randint(2, 48)
        return _case(kind, **heads, seqs=seqs, ctx=_log_int(rng, 1, 1000), rows=rows, kept=rng.randint(1, min(rows, 9)))
    rows = rng.randint(1, 64)
    work = heads["heads"] * heads["head_dim"] * rows * seqs  # queries' values
    return _tree(**heads, seqs=seqs, ctx=_log_int(rng, 1, max(2, min(8000, 30_000_000 // (seqs * per), 1_500_000_000 // work))),
                 rows=rows, type=type_, hidden=rng.choice([0, 0, 50]))


def _lengths(case):
    """History of each sequence of a case, half to one and a half times ``ctx``: the same set for every seed."""
    n = case["seqs"]
    return [case["ctx"]] if n == 1 else [max(1, int(case["ctx"] * (0.5 + (i + 0.5) / n))) for i in range(n)]


def work(case):
    t = SIZE[case.get("type", "float32")]
    if case["kind"] == "score":
        r, n, top = case["rows"], case["n"], case["top"]
        return {"bytes": r * n * t + r * (16 + 8 * top), "flops": 8 * r * n}
    hd, nkv, nh = case["head_dim"], case["kv_heads"], case["heads"]
    ctx = _lengths(case)
    r = case["rows"] * len(ctx)
    if case["kind"] == "keep":  # moved, then read back as float32
        moved = case["kept"] * len(ctx)
        return {"bytes": 2 * moved * nkv * (2 * (hd + 4) + hd + 4 + 4 * hd), "flops": 2 * moved * nkv * hd}
    if case["kind"] == "append":  # written, then read back
        return {"bytes": r * (2 * nh * hd * t + 2 * nkv * (hd * (t + 1) + 4) + 2 * nkv * (hd * (t + 1) + 4)),
                "flops": r * hd * (6 * nh + 10 * nkv)}
    held = sum(c + case["rows"] for c in ctx)
    seen = sum(case["rows"] * (c + 1) for c in ctx)
    return {"bytes": held * nkv * (2 * hd + 8) + 2 * r * nh * hd * t + 4 * r, "flops": 4 * seen * nh * hd}


def _codes(y):
    """Rows of y as codes and float32 scales. In 64 bits: a quotient next to a half goes to one side only."""
    y = y.double()
    scale = (y.abs().amax(-1, keepdim=True) / 127).float()
    scale = torch.where(scale * 127 < 2.0 ** -100, 0.0, scale)
    c = torch.where(scale > 0, torch.round(y / scale.double()), 0.0)
    return c.to(torch.int8), scale.squeeze(-1)


def _frequencies(case):
    """Radians a position of each rotated pair, in 64 bits: theta^(-2 i / rotated), divided by ``scale``; with
    ``original`` only where a turn is long beside it, those in between by how many turns it holds."""
    n = case["rotated"]
    f = case["theta"] ** (-torch.arange(0, n, 2, dtype=torch.float64) / n)
    if case["scale"] == 1.0:
        return f
    if not case["original"]:
        return f / case["scale"]
    turns = case["original"] * f / (2 * math.pi)
    keep = ((turns - 1) / (4 - 1)).clamp(0, 1)
    return keep * f + (1 - keep) * f / case["scale"]


def _tree_of(n, r, g):
    """Parents [n, r] and depths of random trees: nodes hang on one of the few before them, the first ones on the history."""
    back = torch.randint(0, 4, (n, r), generator=g, device=DEV)
    parent = (torch.arange(r, device=DEV) - 1 - back).clamp(min=-1)
    depth = torch.zeros(n, r, dtype=torch.int64, device=DEV)
    for i in range(1, r):
        up = parent[:, i]
        depth[:, i] = torch.where(up >= 0, depth.gather(1, up.clamp(min=0)[:, None])[:, 0] + 1, 0)
    return parent.to(torch.int32), depth.to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    dt = TYPES[case.get("type", "float32")]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    s = {"case": case}
    if case["kind"] == "score":
        r, n = case["rows"], case["n"]
        wide = torch.empty(r, n + case["pad"], dtype=dt, device=DEV)
        for a in range(0, r, 256):  # some rows sure of a few tokens, others not
            x = normal(min(256, r - a), n + case["pad"]) * (1 + 2 * torch.rand(min(256, r - a), 1, generator=g, device=DEV))
            if case["banned"]:
                x.masked_fill_(torch.rand(x.shape, generator=g, device=DEV) * 1000 < case["banned"], -math.inf)
            wide[a:a + 256] = x
        s["logits"] = wide[:, :n]
        likely = torch.stack([x.float().argmax() for x in s["logits"]])
        some = torch.randint(0, n, (r,), generator=g, device=DEV)
        s["target"] = torch.where(torch.rand(r, generator=g, device=DEV) < 0.5, likely, some).to(torch.int32)
        return s
    ctx, r, nkv, nh, hd = _lengths(case), case["rows"], case["kv_heads"], case["heads"], case["head_dim"]
    n, d = len(ctx), -(-hd // PAGE) * PAGE
    order = torch.randperm(n, generator=g, device=DEV).tolist()
    total = [ctx[i] + r for i in order]
    per = [-(-t // PAGE) for t in total]
    pool = sum(per) + 3  # some pages are nobody's
    pages = torch.randperm(pool, generator=g, device=DEV).to(torch.int32)
    s["table"] = torch.zeros(n, max(per), dtype=torch.int32, device=DEV)
    at = 0
    for i, p in enumerate(per):
        s["table"][i, :p] = pages[at:at + p]
        at += p
    s["kv_len"] = torch.tensor(total, dtype=torch.int32, device=DEV)
    s["row_start"] = torch.arange(0, n * r + 1, r, dtype=torch.int32, device=DEV)
    s["rows"], s["most_rows"], s["most_len"] = n * r, r, max(total)
    # the history (and, for attention and what is kept, the drafted rows themselves), as a session left it
    k, k_scale = _codes(normal(pool, nkv, PAGE, hd) * (1 + 3 * (torch.arange(hd, device=DEV) % 16 == 3)))
    v, v_scale = _codes(normal(pool, nkv, PAGE, hd))
    s["keys"] = torch.zeros(pool, nkv, PAGE, d, dtype=torch.int8, device=DEV)
    s["keys"][..., :hd] = k
    s["values"] = torch.zeros(pool, nkv, d, PAGE, dtype=torch.int8, device=DEV)
    s["values"][:, :, :hd] = v.transpose(2, 3)
    s["key_scale"], s["value_scale"] = k_scale, v_scale
    if case["kind"] == "keep":
        # an ascending path of nodes for each sequence, in the places of its first rows: a first few that lie where
        # they belong, then some from behind the places that are filled, so that a pass can be made again
        kept = case["kept"]
        keep = torch.full((n, r), -1, dtype=torch.int32, device=DEV)
        stay = torch.randint(max(0, 2 * kept - r), kept + 1, (n,), generator=g, device=DEV).tolist()
        for i, m in enumerate(stay):
            far = kept + torch.randperm(r - kept, generator=g, device=DEV)[:kept - m].sort().values
            keep[i, :kept] = torch.cat([torch.arange(m, device=DEV), far])
        s["keep"] = keep.reshape(-1)
        s["kept"] = torch.full((n,), kept, dtype=torch.int32, device=DEV)
        s["back_start"] = torch.arange(0, n * kept + 1, kept, dtype=torch.int32, device=DEV)
        return s
    parent, depth = _tree_of(n, r, g)
    if case["kind"] == "tree":
        s["parent"] = parent.reshape(-1)
        s["q"] = normal(n * r, nh, hd).to(dt)
        s["scale"] = 1 / math.sqrt(hd)
        s["hidden"] = None
        if case["hidden"]:
            s["hidden"] = (torch.rand(n, max(total), generator=g, device=DEV) * 1000 < case["hidden"]).to(torch.uint8)
            if n > 2:
                s["hidden"][1] = 1  # a session with nothing to see
        return s
    # queries, keys and values as a fused projection leaves them: slices of wider rows
    y = normal(n * r, (nh + 2 * nkv) * hd).to(dt)
    s["q"] = y[:, :nh * hd].view(n * r, nh, hd)
    s["k"] = y[:, nh * hd:(nh + nkv) * hd].view(n * r, nkv, hd)
    s["v"] = y[:, (nh + nkv) * hd:].view(n * r, nkv, hd)
    s["position"] = None
    if case["tree"]:
        s["position"] = (depth + (s["kv_len"] - r)[:, None]).to(torch.int32).reshape(-1)
    s["q_norm"] = s["k_norm"] = None
    if case["norm"]:
        s["q_norm"], s["k_norm"] = (1 + 0.1 * normal(hd)).to(dt), (1 + 0.1 * normal(hd)).to(dt)
    s["freq"] = _frequencies(case).to(DEV)
    return s


def _positions(start, kv_len, rows):
    """The sequence and the position of each of a call's rows."""
    count = start[1:] - start[:-1]
    seq = torch.repeat_interleave(torch.arange(len(kv_len), device=DEV), count, output_size=rows)
    return seq, (kv_len - count)[seq] + torch.arange(rows, device=DEV) - start[:-1][seq]


def _read(s, start, kv_len, rows, dt):
    """The values of the last positions of each sequence."""
    hd = s["case"]["head_dim"]
    seq, pos = _positions(start, kv_len, rows)
    page, at = s["table"][seq, pos // PAGE].long(), pos % PAGE
    k = s["keys"][page, :, at, :hd] * s["key_scale"][page, :, at][..., None]
    v = s["values"][page, :, :hd, at] * s["value_scale"][page, :, at][..., None]
    return k.to(dt), v.to(dt)


def _rotate(s, x, weight, pos):
    """In 64 bits: far positions' angles, and quotients next to a half once the keys are codes."""
    case, x = s["case"], x.double()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * weight.double()
    n = case["rotated"]
    angle = (pos.double()[:, None] * s["freq"])[:, None]
    c, sn = torch.cos(angle), torch.sin(angle)
    out = x.clone()
    first, second = (slice(0, n, 2), slice(1, n, 2)) if case["interleaved"] else (slice(0, n // 2), slice(n // 2, n))
    out[..., first] = x[..., first] * c - x[..., second] * sn
    out[..., second] = x[..., second] * c + x[..., first] * sn
    return out


def _plain_append(s, dt):
    hd = s["case"]["head_dim"]
    seq, slot = _positions(s["row_start"], s["kv_len"], s["rows"])
    pos = slot if s["position"] is None else s["position"]
    page, at = s["table"][seq, slot // PAGE].long(), slot % PAGE
    codes, scale = _codes(_rotate(s, s["k"], s["k_norm"], pos))
    s["keys"][page, :, at, :hd] = codes
    s["key_scale"][page, :, at] = scale
    codes, scale = _codes(s["v"])
    s["values"][page, :, :hd, at] = codes
    s["value_scale"][page, :, at] = scale
    return (_rotate(s, s["q"], s["q_norm"], pos).to(dt),) + _read(s, s["row_start"], s["kv_len"], s["rows"], dt)


def _plain_tree(s):
    q, n, r = s["q"], len(s["kv_len"]), s["most_rows"]
    nh, hd = q.shape[1:]
    nkv, width = s["keys"].shape[1], s["table"].shape[1]
    long = width * PAGE
    # what each node sees of the tree: its parent's ancestors, its parent, itself
    parent = s["parent"].view(n, r).long()
    sees = torch.eye(r, dtype=torch.bool, device=DEV).expand(n, r, r).clone()
    for i in range(1, r):
        up = parent[:, i]
        above = sees.gather(1, up.clamp(min=0)[:, None, None].expand(n, 1, r))[:, 0]
        sees[:, i] |= above & (up >= 0)[:, None]
    ctx = (s["kv_len"] - r).long()
    at = torch.arange(long, device=DEV)
    node = at[None] - ctx[:, None]                                                   # [n, positions]
    inside = (node >= 0) & (node < r)
    seen = sees.gather(2, node.clamp(0, r - 1)[:, None].expand(n, r, long)) & inside[:, None] | (node < 0)[:, None]
    if s["hidden"] is not None:
        shown = torch.zeros(n, long, dtype=torch.bool, device=DEV)
        shown[:, :s["most_len"]] = s["hidden"] == 0
        seen = seen & shown[:, None]
    out = torch.empty(n, r, nh, hd, device=DEV)
    most = max(1, 400_000_000 // (r * nh * long))
    for a in range(0, n, most):  # some sequences at a time
        table, m = s["table"][a:a + most].long(), min(most, n - a)
        k = s["keys"][table][..., :hd] * s["key_scale"][table][..., None]                # [m, pages, nkv, 64, hd]
        v = s["values"][table][:, :, :, :hd] * s["value_scale"][table][:, :, :, None]    # [m, pages, nkv, hd, 64]
        k = k.permute(0, 2, 4, 1, 3).reshape(m, nkv, hd, long)
        v = v.permute(0, 2, 1, 4, 3).reshape(m, nkv, long, hd)
        wide = q.view(n, r, nkv, nh // nkv, hd)[a:a + most].float().permute(0, 2, 1, 3, 4)
        x = (wide.reshape(m, nkv, -1, hd) @ k).reshape(m, nkv, r, nh // nkv, long) * s["scale"]
        x = torch.where(seen[a:a + most, None, :, None], x, -math.inf)
        top = x.amax(-1, keepdim=True)
        p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
        total = p.sum(-1, keepdim=True)
        o = (p.reshape(m, nkv, -1, long) @ v).reshape(m, nkv, r, nh // nkv, hd)
        o = o / torch.where(total == 0, 1.0, total)
        out[a:a + most] = o.permute(0, 2, 1, 3, 4).reshape(m, r, nh, hd)
    return out.reshape(n * r, nh, hd).to(q.dtype)


def _plain_score(s):
    top, n = s["case"]["top"], s["case"]["n"]
    out = []
    for a in range(0, len(s["target"]), 256):  # some rows at a time
        x, t = s["logits"][a:a + 256].float(), s["target"][a:a + 256].long()[:, None]
        d = x - x.amax(1, keepdim=True)
        e = torch.exp(d)
        total = e.sum(1, keepdim=True, dtype=torch.float64)
        log_total = torch.log(total)
        entropy = log_total - (torch.where(e > 0, d, 0.0) * e).sum(1, keepdim=True, dtype=torch.float64) / total
        log_p = (d.gather(1, t) - log_total).float()[:, 0]
        rank = (x > x.gather(1, t)).sum(1)
        # value first, then the lower index: a whole number that orders both
        bits = (x + 0.0).view(torch.int32)
        bits = (bits ^ ((bits >> 31) & 0x7fffffff)).long()
        index = (bits * 2 ** 32 + (2 ** 32 - 1 - torch.arange(n, device=DEV))).topk(top, 1).indices
        out.append((log_p, entropy.float()[:, 0], rank.to(torch.int32), index.to(torch.int32),
                    (d.gather(1, index) - log_total).float()))
    return tuple(torch.cat(part) for part in zip(*out))


def _plain_keep(s):
    case = s["case"]
    r, hd = case["rows"], case["head_dim"]
    ctx = (s["kv_len"] - r).long()[:, None]
    new, old = ctx + torch.arange(case["kept"], device=DEV), ctx + s["keep"].view(-1, r)[:, :case["kept"]]
    seq = torch.arange(len(ctx), device=DEV)[:, None]
    to, to_at = s["table"][seq, new // PAGE].long(), new % PAGE
    page, at = s["table"][seq, old // PAGE].long(), old % PAGE
    s["keys"][to, :, to_at], s["key_scale"][to, :, to_at] = s["keys"][page, :, at], s["key_scale"][page, :, at]
    s["values"][to, :, :hd, to_at], s["value_scale"][to, :, to_at] = s["values"][page, :, :hd, at], s["value_scale"][page, :, at]
    kv_len = s["kv_len"] - r + s["kept"]
    return (kv_len,) + _read(s, s["back_start"], kv_len, len(ctx) * case["kept"], torch.float32)


def run(s):
    case = s["case"]
    dt = TYPES[case.get("type", "float32")]
    if not own:
        if case["kind"] == "append":
            return _plain_append(s, dt)
        if case["kind"] == "tree":
            return _plain_tree(s)
        if case["kind"] == "score":
            return _plain_score(s)
        return _plain_keep(s)
    from defer_amd import q8

    if case["kind"] == "score":
        return tuple(q8.log_probs(s["logits"], s["target"], top=case["top"]))
    pages = q8.Pages(s["keys"], s["values"], s["key_scale"], s["value_scale"], s["table"])
    if case["kind"] == "append":
        q = q8.kv_append(pages, s["q"], s["k"], s["v"], s["kv_len"], q8.Rotary(s["freq"], case["interleaved"]), s["row_start"],
                         most_rows=s["most_rows"], position=s["position"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=1e-6)
        return (q,) + q8.kv_read(pages, s["kv_len"], s["row_start"], s["rows"], case["head_dim"], most_rows=s["most_rows"],
                                 dtype=dt)
    if case["kind"] == "tree":
        return q8.tree_attention(s["q"], pages, s["parent"], s["kv_len"], s["row_start"], most_rows=s["most_rows"],
                                 most_len=s["most_len"], scale=s["scale"], hidden=s["hidden"])
    kv_len = q8.kv_keep(pages, s["kv_len"], s["row_start"], s["keep"], s["kept"], most_rows=s["most_rows"])
    return (kv_len,) + q8.kv_read(pages, kv_len, s["back_start"], case["seqs"] * case["kept"], case["head_dim"],
                                  most_rows=case["kept"])


def exact(case, seed):
    """The operators' definitions in 64 bits, a row, or a sequence and a head, at a time."""
    s = prepare(case, seed)
    f = torch.float64
    if case["kind"] == "score":
        out = []
        for x, t in zip(s["logits"], s["target"].tolist()):
            x = x.to(f)
            log_z = torch.logsumexp(x, 0)
            lp = x - log_z
            order = torch.sort(x, descending=True, stable=True).indices[:case["top"]]
            out.append((lp[t], -torch.nansum(torch.exp(lp) * lp), (x > x[t]).sum().to(torch.int32), order.to(torch.int32),
                        lp[order]))
        return tuple(torch.stack(part) for part in zip(*out))
    hd, n, r = case["head_dim"], case["seqs"], case["rows"]
    lens = s["kv_len"].tolist()

    def held(i):
        """Keys and values of sequence i, position by position: [positions, heads, head size]."""
        p = s["table"][i, :-(-lens[i] // PAGE)].long()
        k = s["keys"][p].to(f) * s["key_scale"][p].to(f).unsqueeze(3)
        v = s["values"][p].to(f) * s["value_scale"][p].to(f).unsqueeze(2)
        k, v = k.transpose(1, 2).flatten(0, 1), v.permute(0, 3, 1, 2).flatten(0, 1)
        return k[:lens[i], :, :hd], v[:lens[i], :, :hd]

    if case["kind"] == "keep":
        ks, vs = [], []
        for i in range(n):
            k, v = held(i)
            at = lens[i] - r + s["keep"][i * r:i * r + case["kept"]].long()
            ks.append(k[at])
            vs.append(v[at])
        return s["kv_len"] - r + case["kept"], torch.cat(ks), torch.cat(vs)
    if case["kind"] == "append":
        pos = torch.cat([torch.arange(m - r, m, device=DEV) for m in lens]) if s["position"] is None else s["position"]
        turn = torch.polar(torch.ones((), dtype=f, device=DEV), pos.to(f)[:, None] * s["freq"])[:, None]

        def turned(x, w):
            x = x.to(f)
            if w is not None:
                x = x * w.to(f) / torch.sqrt((x * x).sum(-1, keepdim=True) / hd + 1e-6)
            m = case["rotated"]
            pairs = x[..., :m].unflatten(-1, (-1, 2) if case["interleaved"] else (2, -1))
            pairs = pairs if case["interleaved"] else pairs.transpose(-1, -2)
            z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
            z = z if case["interleaved"] else z.transpose(-1, -2)
            return torch.cat([z.flatten(-2), x[..., m:]], -1)

        def coded(y):
            step = (y.abs().max(-1, keepdim=True).values / 127).float().to(f)
            return torch.round(y / step) * step

        return turned(s["q"], s["q_norm"]), coded(turned(s["k"], s["k_norm"])), coded(s["v"].to(f))
    out = torch.zeros(n * r, case["heads"], hd, dtype=f, device=DEV)
    parent, group = s["parent"].tolist(), case["heads"] // case["kv_heads"]
    for i in range(n):
        k, v = held(i)
        off = torch.ones(r, lens[i], dtype=torch.bool)
        off[:, :lens[i] - r] = False
        for j in range(r):
            at = j
            while at >= 0:
                off[j, lens[i] - r + at] = False
                at = parent[i * r + at]
        off = off.to(DEV)
        if s["hidden"] is not None:
            off = off | (s["hidden"][i, :lens[i]] != 0)[None, :]
        for h in range(case["heads"]):
            x = torch.matmul(s["q"][i * r:(i + 1) * r, h].to(f), k[:, h // group].t()) * s["scale"]
            x = torch.softmax(x.masked_fill(off, -math.inf), 1)
            out[i * r:(i + 1) * r, h] = torch.matmul(torch.nan_to_num(x, nan=0.0), v[:, h // group])
    return out
