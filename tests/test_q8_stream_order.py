"""Host path of a model in 8 bits, over the stand-in for the HIP runtime that
test_stream_order.py describes: what it queues is ordered, a call that fails
leaves nothing running, and what it does not do it refuses."""
import ctypes
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("fake") / "libfake_hip.so")
    subprocess.run(["gcc", "-O1", "-Wall", "-shared", "-fPIC", "-I/opt/rocm/include", "-o", out,
                    os.path.join(ROOT, "tests", "probe", "fake_hip.c")], check=True)
    return out


@pytest.mark.parametrize("check", ["order", "failure", "refusals"])
def test_host_path(fake, check):
    r = subprocess.run([sys.executable, os.path.abspath(__file__), fake, check], cwd=ROOT,
                       env=dict(os.environ, PYTHONPATH=ROOT), capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
    assert r.stdout.strip().endswith("ok"), r.stdout + r.stderr


def check_order(hip, G, m, cfg, w):
    c = m.new_cache(64)
    m.prompt(c, list(range(20)))
    calls = {
        "forward": lambda x: m.forward(1, x),
        "masked forward": lambda x: m.forward(1, x, masked=[2]),
        "truncate + forward": lambda x: (x.truncate(10), m.forward(1, x)),
        "prompt": lambda x: m.prompt(x, [3] * 20),
        "short prompt": lambda x: m.prompt(x, [3]),
        "forward_batch": lambda x: m.forward_batch([x, m.new_cache(64), x], [1, 2, 3], logits=True),
        "step_batch": lambda x: m.step_batch([x, c], 0.7, [1, 2]),
        "generate": lambda x: m.generate(x, 2, 0.7, [1, 2], stop=[4]),
        "read": lambda x: x.read(1),
        "set_logits": lambda x: x.set_logits([0.0] * cfg["vocab_size"]),
        "replay": lambda x: m.replay(m.new_cache(64), [1, 2, 3, 4], 2, 0.7, [1, 2]),
        "a new model": lambda x: G.GpuModel(m.cfg, w, bits=8).new_cache(8).clone(),
    }
    bad = []
    for name, call in calls.items():
        before = hip.fake_unordered()
        x = c.clone()
        if hip.fake_pending():
            bad.append("clone, unfinished on return, before " + name)
        call(x)
        if hip.fake_unordered() != before:
            bad.append(name)
        x.close()
    assert not bad, bad


def check_failure(hip, G, m, cfg, w):
    calls = {
        "forward": lambda a, b: m.forward(1, a, masked=[3]),
        "forward_batch": lambda a, b: m.forward_batch([a, b], [1, 2], logits=True),
        "read": lambda a, b: a.read(0),
        "generate": lambda a, b: m.generate(a, 2, 0.5, [1, 2]),
    }
    bad = []
    for name, call in calls.items():
        for k in range(3):
            a, b = m.new_cache(64), m.new_cache(64)
            for c in (a, b):
                m.prompt(c, list(range(20)))
            hip.fake_fail_in(k + 1)
            try:
                call(a, b)
                bad.append((name, k, "no error"))
            except G.DeferGpuError:
                pass
            hip.fake_fail_in(0)
            if hip.fake_pending():
                bad.append((name, k, "still running"))
            assert len(a) == 20
            m.forward(1, a)  # a mask that was not used does not stay behind
            a.close()
            b.close()
    assert not bad, bad


def check_refusals(hip, G, m, cfg, w):
    c = m.new_cache(30)
    m.prompt(c, [1, 2, 3])

    def refused(code, call):
        try:
            call()
        except G.DeferGpuError as e:
            assert e.code == code, e
            return
        raise AssertionError("not refused")

    refused(G.E_INVALID, lambda: m.forward(1, c, trace=True))
    refused(G.E_INVALID, lambda: c.value_norms(0, 1))
    refused(G.E_INVALID, lambda: m.generate_static(c, 2, 0.0))
    refused(G.E_TOKEN, lambda: m.forward(cfg["vocab_size"], c))
    refused(G.E_TOKEN, lambda: m.forward_batch([c], [cfg["vocab_size"]]))
    refused(G.E_CONTEXT, lambda: m.prompt(c, [1] * 28))
    assert len(c) == 30
    refused(G.E_CONTEXT, lambda: m.forward(1, c))
    refused(G.E_CONTEXT, lambda: m.generate(c, 1, 0.0))
    refused(G.E_NO_LOGITS, lambda: m.generate(m.new_cache(8), 1, 0.0))
    refused(G.E_NO_LOGITS, lambda: m.step(m.new_cache(8), 0.0))
    m.prompt(m.new_cache(8), [])
    assert m.replay(m.new_cache(8), [], 0, 0.0) == (-1, 0)
    # another model's cache, and flags that are none
    other = G.GpuModel(m.cfg, w)
    refused(G.E_INVALID, lambda: other.forward(1, c))
    ptrs = (ctypes.c_void_p * len(w))(*[a.ctypes.data for a in w])
    out = ctypes.c_void_p()
    assert G.lib().defer_gpu_model_create(ctypes.byref(m.cfg), ptrs, len(w), 2, ctypes.byref(out)) == G.E_INVALID
    assert not out.value
    try:
        G.GpuModel(m.cfg, w, bits=4)
        raise AssertionError("not refused")
    except ValueError:
        pass


if __name__ == "__main__":
    hip = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)  # found before the real runtime
    hip.fake_unordered.restype = ctypes.c_long
    from defer_amd import gpu as G
    from defer_amd import synthetic

    cfg = synthetic.CONFIGS["tiny"]
    weights = synthetic.make_weights(cfg, 1)
    model = G.GpuModel(G.Config.from_dict(cfg), weights, bits=8)
    {"order": check_order, "failure": check_failure, "refusals": check_refusals}[sys.argv[2]](hip, G, model, cfg, weights)
    print("ok")
