"""The package imports on a torch build that has no GPU bindings (a build for the CPU alone)."""
import os
import pkgutil
import subprocess
import sys

import lockstep_amd

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_every_module_imports_without_torchs_gpu_bindings():
    names = [m.name for m in pkgutil.iter_modules(lockstep_amd.__path__, "lockstep_amd.")
             if not m.name.split(".")[-1].startswith("lib")]   # (the shared library itself)
    code = ("import importlib, torch\n"
            "for n in ('_cuda_getDevice', '_cuda_getCurrentRawStream'):\n"
            "    if hasattr(torch._C, n):\n"
            "        delattr(torch._C, n)\n"
            "for n in %r:\n"
            "    importlib.import_module(n)\n" % (names,))
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
