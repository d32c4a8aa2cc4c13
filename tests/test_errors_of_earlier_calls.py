"""An error is told once, to the call that met it: not again by the next call's
launches, which ask the runtime how they went. Over the stand-in for the HIP
runtime that test_stream_order.py describes, with the runtime's last error and
allocations that fail added."""
import ctypes
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

FAKE = r"""
#define hipMalloc plain_malloc
#define hipGetLastError plain_get_last_error
#include "fake_hip.c"
#undef hipMalloc
#undef hipGetLastError

static hipError_t last;
static int fail_malloc;
void fake_fail_malloc_in(int n) { fail_malloc = n; }
void fake_set_last(int e) { last = (hipError_t)e; }
int fake_last(void) { return last; }

hipError_t hipMalloc(void** p, size_t n) {
  if (fail_malloc > 0 && --fail_malloc == 0) return last = hipErrorOutOfMemory;
  return plain_malloc(p, n);
}
hipError_t hipGetLastError(void) {
  const hipError_t e = last;
  last = hipSuccess;
  return e;
}
"""


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    d = tmp_path_factory.mktemp("fake")
    (d / "fake.c").write_text(FAKE)
    out = str(d / "libfake_hip.so")
    subprocess.run(["gcc", "-O1", "-Wall", "-shared", "-fPIC", "-I/opt/rocm/include", "-I", os.path.join(ROOT, "tests", "probe"),
                    "-o", out, str(d / "fake.c")], check=True)
    return out


@pytest.mark.parametrize("check", ["own", "foreign"])
def test_an_error_is_told_once(fake, check):
    r = subprocess.run([sys.executable, os.path.abspath(__file__), fake, check], cwd=ROOT,
                       env=dict(os.environ, PYTHONPATH=ROOT), capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
    assert r.stdout.strip().endswith("ok"), r.stdout + r.stderr


def check_own(hip, G, q8, cfg, w):
    """A cache that there is no memory for, then calls on what is there."""
    c = G.Config.from_dict(cfg)
    for bits in (32, 8):
        m = G.GpuModel(c, w, bits=bits)
        calls = {
            "prompt": lambda x: m.prompt(x, [3] * 20),
            "read": lambda x: (m.prompt(x, [1, 2, 3]), x.read(0)),
            "clone": lambda x: x.clone(),
            "quantize": lambda x: _quantize(q8),
        }
        if bits == 8:  # (the stand-in runs no kernel that a single f32 token's call could wait for)
            calls["forward"] = lambda x: m.forward(1, x)
        for name, call in calls.items():
            for k in (1, 2, 3):
                x = m.new_cache(64)
                hip.fake_fail_malloc_in(k)
                try:
                    m.new_cache(64)
                    raise AssertionError("no error")
                except G.DeferGpuError as e:
                    assert e.code == G.E_HIP, e
                hip.fake_fail_malloc_in(0)
                assert hip.fake_last() == 0, (name, k)
                call(x)
                x.close()
        hip.fake_fail_malloc_in(1)
        try:
            G.GpuModel(c, w, bits=bits)
            raise AssertionError("no error")
        except G.DeferGpuError:
            pass
        hip.fake_fail_malloc_in(0)
        assert hip.fake_last() == 0


def _quantize(q8):
    P = 4096
    assert q8._lib().defer_gpu_q8_quantize(0, P, 64, 2, 64, P, P, None) == 0


def check_foreign(hip, G, q8, cfg, w):
    """The program's own error stays there for it."""
    P, L = 4096, q8._lib()
    pages, rows = q8._CPages(P, P, P, P, P, 4, 2, 64, 2), q8._CRows(P, P, 2, 5, 3)
    none = q8._CRows(P, P, 2, 5, 0)
    calls = {
        "quantize": lambda: _quantize(q8),
        "rms_norm": lambda: L.defer_gpu_q8_rms_norm(0, P, 64, None, 0, P, 1e-5, 2, 64, None, 0, P, P, None),
        "linear": lambda: L.defer_gpu_q8_linear(P, 64, P, P, 64, P, 2, 64, 64, 0, P, 64, None),
        "linear, many rows": lambda: L.defer_gpu_q8_linear(P, 64, P, P, 64, P, 500, 640, 64, 0, P, 640, None),
        "linear, unaligned": lambda: L.defer_gpu_q8_linear(P, 63, P, P, 63, P, 1000, 2000, 63, 0, P, 2000, None),
        "kv_write": lambda: L.defer_gpu_q8_kv_write(pages, rows, 0, P, 128, P, 128, None),
        "kv_read": lambda: L.defer_gpu_q8_kv_read(pages, rows, 0, P, P, None),
        "kv_read of nothing": lambda: L.defer_gpu_q8_kv_read(pages, none, 0, P, P, None),
        "attention": lambda: L.defer_gpu_q8_attention(pages, rows, 0, P, 256, 4, 128, 1.0, None, 0, 0, P, 256, 0, P, 1 << 20, None),
        "attention, split": lambda: L.defer_gpu_q8_attention(pages, rows, 0, P, 256, 4, 6000, 1.0, None, 0, 0, P, 256, 0, P, 1 << 24, None),
        "attention to nothing": lambda: L.defer_gpu_q8_attention(pages, none, 0, P, 256, 4, 128, 1.0, None, 0, 0, P, 256, 1, P, 1 << 20, None),
    }
    for name, call in calls.items():
        hip.fake_set_last(2)
        assert call() in (0, None), (name, G.lib().defer_gpu_last_error())
        assert hip.fake_last() == 2, name


if __name__ == "__main__":
    hip = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)  # found before the real runtime
    from defer_amd import gpu as G
    from defer_amd import q8, synthetic

    cfg = synthetic.CONFIGS["tiny"]
    weights = synthetic.make_weights(cfg, 1)
    {"own": check_own, "foreign": check_foreign}[sys.argv[2]](hip, G, q8, cfg, weights)
    print("ok")
