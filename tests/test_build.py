"""The build where torch is not installed: all but what is made of torch."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CODE = r"""
import sys

class NoTorch:
    def find_spec(self, name, path=None, target=None):
        if name == "torch":
            raise ModuleNotFoundError("No module named 'torch'", name="torch")

WITHOUT = sys.argv[1] == "without"
if WITHOUT:
    import importlib.util
    real = importlib.util.find_spec
    importlib.util.find_spec = lambda name, package=None: None if name == "torch" else real(name, package)
    sys.meta_path.insert(0, NoTorch())

import __graft_entry__ as entry
from defer_amd import build as B

ran = []
B.PKG = B.BUILD = sys.argv[2]  # nothing of what is built is touched
B._run = lambda cmd, cwd=None: ran.append(" ".join(cmd))
B.os.replace = lambda a, b: None
entry.subprocess.run = lambda cmd, **kw: ran.append(" ".join(cmd))
entry.build()
for what in ("libdefer_gpu.so", "libdefer_gpu.a", "libdefer_host.so", "abi_test", "libexact_probe.so", "oracle"):
    assert any(what in r for r in ran), what
assert any("_q8_torch.so" in r for r in ran) == (not WITHOUT)
assert ("torch" in sys.modules) == (not WITHOUT)
print("ok")
"""


def run(which, tmp):
    r = subprocess.run([sys.executable, "-c", CODE, which, str(tmp)], cwd=ROOT, env=dict(os.environ, PYTHONPATH=ROOT), capture_output=True,
                       text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip().endswith("ok"), r.stdout + r.stderr


def test_build_without_torch(tmp_path):
    run("without", tmp_path)


def test_build_with_torch(tmp_path):
    run("with", tmp_path)
