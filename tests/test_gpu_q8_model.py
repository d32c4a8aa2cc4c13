"""GPU: a model in 8 bits (DEFER_GPU_MODEL_8BIT): its forwards against 64-bit
formulas that round to codes at the same places, the same bits however rows are
grouped into calls, and the session calls -- generate, lockstep, checkout,
clone, truncation, masks -- on it."""
import numpy as np
import pytest

from defer_amd import gpu as G
from defer_amd import host as H
from defer_amd import synthetic

pytestmark = pytest.mark.gpu


def bits(a):
    return np.ascontiguousarray(a, dtype=np.float32).view(np.uint32)


def codes(y):
    """What rows of y stand for in 8 bits, in 64 bits."""
    top = np.abs(y).max(-1, keepdims=True)
    s = (top / 127).astype(np.float32).astype(np.float64)
    return np.where(top < 2.0 ** -100, 0.0, np.rint(np.divide(y, s, out=np.zeros_like(y), where=s > 0)) * s)


class Formula:
    """One session of the model, a token at a time, in 64 bits."""

    def __init__(self, cfg, w):
        self.c = cfg
        t = [np.asarray(x, dtype=np.float64) for x in w]
        k = iter(t)
        self.embed = next(k)
        self.layers = []
        for _ in range(cfg["num_layers"]):
            names = ["an", "wq"] + ["bq"] * cfg["has_bias"] + ["wk"] + ["bk"] * cfg["has_bias"] + ["wv"] + \
                    ["bv"] * cfg["has_bias"] + ["wo", "fn", "wg", "wu", "wd"]
            d = {n: next(k) for n in names}
            for n in names:
                if n[0] == "w":
                    d[n] = codes(d[n])
            self.layers.append(d)
        self.norm = next(k)
        self.head = codes(self.embed if cfg["tie_word_embeddings"] else next(k))
        self.k = [[] for _ in self.layers]
        self.v = [[] for _ in self.layers]

    def rms(self, x, w):
        return codes((x / np.sqrt(np.mean(x * x) + float(np.float32(self.c["rms_norm_eps"]))) * w)[None])[0]

    def rope(self, x, pos):
        half = self.c["head_dim"] // 2
        inv = (1.0 / float(np.float32(self.c["rope_theta"])) ** (np.arange(half) * 2.0 / self.c["head_dim"])).astype(np.float32)
        a = (np.float32(pos) * inv).astype(np.float64)
        x0, x1 = x[:, :half], x[:, half:]
        return np.concatenate([x0 * np.cos(a) - x1 * np.sin(a), x1 * np.cos(a) + x0 * np.sin(a)], 1)

    def forward(self, token, masked=()):
        c = self.c
        nh, nkv, hd = c["num_heads"], c["num_kv_heads"], c["head_dim"]
        x = self.embed[token].copy()
        pos = len(self.k[0])
        for l, W in enumerate(self.layers):
            y = self.rms(x, W["an"])
            q, k, v = (W[n] @ y + W.get("b" + n[1], 0.0) for n in ("wq", "wk", "wv"))
            self.k[l].append(codes(self.rope(k.reshape(nkv, hd), pos)))
            self.v[l].append(codes(v.reshape(nkv, hd)))
            q = self.rope(q.reshape(nh, hd), pos)
            kk, vv = np.stack(self.k[l]), np.stack(self.v[l])
            s = np.einsum("hd,thd->ht", q, kk.repeat(nh // nkv, 1)) / np.sqrt(hd)
            s[:, [t for t in masked if t < pos]] = -np.inf
            p = np.exp(s - s.max(1, keepdims=True))
            o = np.einsum("ht,thd->hd", p / p.sum(1, keepdims=True), vv.repeat(nh // nkv, 1))
            x = x + W["wo"] @ codes(o.reshape(1, -1))[0]
            y = self.rms(x, W["fn"])
            g, u = W["wg"] @ y, W["wu"] @ y
            a = g / (1 + np.exp(-g)) if c["activation"] == 0 else \
                0.5 * g * (1 + np.tanh(0.7978846 * (g + 0.044715 * g ** 3)))
            x = x + W["wd"] @ codes((a * u)[None])[0]
        return self.head @ self.rms(x, self.norm)


def model(shape="tiny", seed=5, std=0.08, **kw):
    cfg = dict(synthetic.CONFIGS[shape], **kw)
    w = synthetic.make_weights(cfg, seed, std=std)
    g = np.random.default_rng(seed)
    w = [a if a.ndim == 2 else (a + g.normal(0, 0.1, a.shape)).astype(np.float32) for a in w]  # norms and biases of their own
    return cfg, w, G.GpuModel(G.Config.from_dict(cfg), w, bits=8)


@pytest.fixture(scope="module")
def tiny():
    return model()


def near(got, want):
    """f32 against 64 bits, between them the codes: where no quotient lies within an
    f32 rounding of a half, every code is the same and the logits are off by f32
    roundings only -- of sums of ~100 terms through two layers, far under 2^-24 *
    2000 = 1.2e-4 of the largest. Where one does (about 900 codes a token, each
    moved with a probability of about 1e-5 by an error of 1e-6 of a step's
    half), a code is one step off: max / 127 of its row, which reaches the logits
    as at most a few such steps: 5 % of the largest bounds it."""
    e = np.abs(got - want).max() / np.abs(want).max()
    assert e < 0.05, e
    return e < 1.2e-4


@pytest.mark.parametrize("kw", [{}, {"activation": 1, "has_bias": 1}, {"tie_word_embeddings": 1, "num_kv_heads": 1},
                                {"head_dim": 32, "num_kv_heads": 4, "intermediate_size": 100}])
def test_forward_against_the_formulas(kw):
    cfg, w, m = model(**kw)
    f, c = Formula(cfg, w), m.new_cache(160)
    toks = synthetic.make_prompt(cfg["vocab_size"], 140, seed=1)
    tight = 0
    for i, t in enumerate(toks):
        got = m.forward(int(t), c)
        want = f.forward(int(t))
        tight += near(got, want)
        if i in (0, 70, 139):
            for l in range(cfg["num_layers"]):
                k, v = c.read(l)
                kk, vv = np.stack(f.k[l]).reshape(i + 1, -1), np.stack(f.v[l]).reshape(i + 1, -1)
                # a moved code is one step, 1/127 of its head's largest value
                assert np.abs(k - kk).max() <= np.abs(kk).max() / 50 and np.abs(v - vv).max() <= np.abs(vv).max() / 50
                assert (np.abs(k - kk) > 1e-5).mean() < 0.01 and (np.abs(v - vv) > 1e-5).mean() < 0.01
    # a moved code stays in the cache, so that later rows may see it: most rows see none
    assert tight >= 0.5 * len(toks), tight


def test_masked_forward_against_the_formulas(tiny):
    cfg, w, m = tiny
    toks = [int(t) for t in synthetic.make_prompt(cfg["vocab_size"], 30, seed=2)]
    f, c = Formula(cfg, w), m.new_cache(64)
    for t in toks[:-1]:
        f.forward(t)
    m.prompt(c, toks[:-1])
    masked = [0, 3, 4, 11, 28, 29, 500]  # its own position and later ones are ignored
    base = c.clone()
    got = m.forward(toks[-1], c, masked=masked)
    near(got, f.forward(toks[-1], masked=masked))
    plain = m.forward(toks[-1], base.clone())
    assert np.abs(got - plain).max() > 1e-3
    assert np.array_equal(bits(m.forward(toks[-1], base.clone(), masked=[29, 40])), bits(plain))
    assert np.array_equal(bits(m.forward(toks[-1], base, masked=masked)), bits(got))
    # the next forward sees them again
    assert np.array_equal(bits(m.forward(1, base)), bits(m.forward(1, c)))


@pytest.mark.parametrize("shape,n", [("tiny", 300), ("smollm2-135m", 150)])
def test_rows_are_the_same_however_they_are_grouped(shape, n):
    cfg, w, m = model(shape, std=0.02)
    toks = [int(t) for t in synthetic.make_prompt(cfg["vocab_size"], n, seed=3)]
    one = m.new_cache(n + 8)
    logits = np.stack([m.forward(t, one) for t in toks])
    at_once = m.new_cache(n + 8)
    m.prompt(at_once, toks)
    assert np.array_equal(bits(at_once.last_logits()), bits(logits[-1]))
    for l in range(cfg["num_layers"]):
        for a, b in zip(one.read(l), at_once.read(l)):
            assert np.array_equal(bits(a), bits(b))
    batch = m.new_cache(n + 8)
    assert np.array_equal(bits(m.forward_batch([batch] * n, toks, logits=True)), bits(logits))
    # sessions of other lengths in between, one of them listed twice and apart
    a, b, c = m.new_cache(n + 8), m.new_cache(n + 8), m.new_cache(n + 8)
    m.prompt(a, toks[:70])
    m.prompt(b, toks[:3])
    got = m.forward_batch([a, b, a, c, b, b], [toks[70], toks[3], toks[71], toks[0], toks[4], toks[5]], logits=True)
    for row, i in enumerate((70, 3, 71, 0, 4, 5)):
        assert np.array_equal(bits(got[row]), bits(logits[i])), row
    assert len(a) == 72 and len(b) == 6 and len(c) == 1
    # a truncated cache goes on as if it had never been longer
    at_once.truncate(65)
    m.prompt(at_once, toks[65:100])
    assert np.array_equal(bits(at_once.last_logits()), bits(logits[99]))


def test_generate_steps_lockstep_and_stop(tiny):
    cfg, w, m = tiny
    prompt = [int(t) for t in synthetic.make_prompt(cfg["vocab_size"], 20, seed=4)]
    words = np.random.default_rng(1).integers(0, 1 << 32, 40, dtype=np.uint32)
    for T in (0.0, 0.9):
        c = m.new_cache(100)
        m.prompt(c, prompt)
        toks = m.generate(c, 40, T, words)
        assert len(toks) == 40 and len(c) == 60
        s, x = m.new_cache(100), m.new_cache(100)
        m.prompt(s, prompt)
        m.prompt(x, prompt[:5])
        for i, t in enumerate(toks):
            if i % 3 == 0:
                assert m.sample(s, T, int(words[i])) == t
            if i % 2:
                assert m.step(s, T, int(words[i])) == t
            else:
                assert m.step_batch([x, s], T, [7, words[i]])[1] == t
        assert np.array_equal(bits(s.last_logits()), bits(c.last_logits()))
        if T == 0:
            assert toks[0] == int(np.argmax(_logits(m, prompt)))
        # a stop token ends the run once it has been fed; the callback sees every token
        stop = toks[6]
        e, seen = m.new_cache(100), []
        m.prompt(e, prompt)
        assert m.generate_cb(e, 40, T, words, stop=[stop], on_token=lambda i, t: seen.append((i, t))) == toks[:toks.index(stop) + 1]
        assert seen == list(enumerate(toks[:toks.index(stop) + 1])) and len(e) == 20 + len(seen)
        e = m.new_cache(100)
        m.prompt(e, prompt)
        with pytest.raises(G.DeferGpuError) as err:
            m.generate_cb(e, 40, T, words, on_token=lambda i, t: 3 if i == 4 else 0)
        assert err.value.code == G.E_CALLBACK and m.last_n == 5 and len(e) == 25
        full = m.new_cache(23)
        m.prompt(full, prompt)
        with pytest.raises(G.DeferGpuError) as err:
            m.generate(full, 10, T, words)
        assert err.value.code == G.E_CONTEXT and len(full) == 23


def _logits(m, toks):
    c = m.new_cache(len(toks))
    m.prompt(c, toks)
    return c.last_logits()


def test_session_and_checkout(tiny):
    cfg, w, m = tiny
    prompt = [int(t) for t in synthetic.make_prompt(cfg["vocab_size"], 33, seed=5)]
    s = H.Session(m, H.seed_from_u64(9), 0.8)
    s.prompt(prompt)
    toks = s.generate(120)
    assert len(toks) == 120
    again = H.Session(m, H.seed_from_u64(9), 0.8)
    again.prompt(prompt)
    assert again.generate(120) == toks
    # a recorded session is verified in one batch, a changed one is found where it changed
    r = np.random.default_rng(3).integers(0, 1 << 32, 100, dtype=np.uint32)
    c = m.new_cache(200)
    m.prompt(c, prompt)
    out = m.generate(c, 100, 0.8, r)
    f = m.new_cache(200)
    assert m.replay(f, prompt + out, len(prompt), 0.8, r) == (-1, 0)
    assert np.array_equal(bits(f.last_logits()), bits(c.last_logits())) and len(f) == 133
    assert H.cache_fingerprint(f) == H.cache_fingerprint(c)
    bad = list(out)
    bad[60] = (bad[60] + 1) % cfg["vocab_size"]
    f = m.new_cache(200)
    assert m.replay(f, prompt + bad, len(prompt), 0.8, r) == (len(prompt) + 60, out[60])
    assert len(f) == len(prompt) + 60


def test_clone_is_apart_from_its_source(tiny):
    cfg, w, m = tiny
    toks = [int(t) for t in synthetic.make_prompt(cfg["vocab_size"], 80, seed=6)]
    a = m.new_cache(100)
    m.prompt(a, toks[:70])
    b = a.clone()
    m.prompt(b, toks[70:])
    other = m.new_cache(100)
    m.prompt(other, toks[:70] + [1, 2, 3])
    m.prompt(a, [1, 2, 3])
    assert np.array_equal(bits(a.last_logits()), bits(other.last_logits()))
    assert np.array_equal(bits(b.last_logits()), bits(_logits(m, toks)))


def test_near_the_f32_model():
    """8 bits against f32 on the same weights: how far the roundings carry at the
    135M shape. A code's step is max / 127, with max about 4 of a row's rms: an rms
    error of 4 / 127 / sqrt(12) = 0.9 % in each of a product's two inputs, 1.3 % of
    its output; 210 products (7 x 30) in a row, were all of it to add up in the
    residual, 1.3 % * sqrt(210) = 19 %. The logits are within that of f32's."""
    cfg = synthetic.CONFIGS["smollm2-135m"]
    w = synthetic.make_weights(cfg, 0)
    toks = synthetic.make_prompt(cfg["vocab_size"], 40, seed=1)
    a, b = G.GpuModel(G.Config.from_dict(cfg), w), G.GpuModel(G.Config.from_dict(cfg), w, bits=8)
    x, y = _logits(a, toks), _logits(b, toks)
    assert np.linalg.norm(x - y) / np.linalg.norm(x) < 0.19


def test_profiling_and_settings_change_nothing(tiny):
    cfg, w, _ = tiny
    m = G.GpuModel(G.Config.from_dict(cfg), w, bits=8)
    m.set_grid(3, 5)
    m.set_exec(G.EXEC_GRAPH)
    m.set_batching(0)
    toks = [int(t) for t in synthetic.make_prompt(cfg["vocab_size"], 50, seed=7)]
    want = _logits(tiny[2], toks)
    assert np.array_equal(bits(_logits(m, toks)), bits(want))
    m.set_profiling(True)
    assert np.array_equal(bits(_logits(m, toks)), bits(want))
    st = m.batch_stats()
    assert st["gemm_launches"] == 4 * cfg["num_layers"] + 1 and st["attn_launches"] == cfg["num_layers"]
