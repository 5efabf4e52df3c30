"""The build of the native host path: the library does without it, and it serves the torch it was
compiled against alone."""
import os
import subprocess
import sys

import torch

from conftest import ROOT
from rocketllm_b200 import kernels
from rocketllm_b200.csrc import build


def python(code):
    return subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True,
                          env={**os.environ, "PYTHONPATH": ROOT})


def test_the_library_builds_without_torch_headers_or_a_host_compiler():
    """Up to date here, so that the library itself needs no compiler for this."""
    build.build()
    p = python("import sys; sys.modules['torch'] = None\n"
               "import runpy; m = runpy.run_path('rocketllm_b200/csrc/build.py')\n"
               "assert m['native_missing']() == ['torch']\n"
               "print(m['build']())")
    assert p.returncode == 0, p.stderr
    assert "left out: no torch" in p.stdout and p.stdout.split()[-1] == build.LIB
    p = python("import os, runpy\n"
               "m = runpy.run_path('rocketllm_b200/csrc/build.py'); os.environ['PATH'] = ''\n"
               "m['build_native'](force=True)")
    assert p.returncode == 0 and "left out: no g++" in p.stdout, p.stderr


def test_another_torch_or_python_means_another_build(monkeypatch, tmp_path):
    ran = []
    monkeypatch.setattr(build, "NATIVE_STAMP", str(tmp_path / "against"))
    monkeypatch.setattr(build.subprocess, "run", lambda cmd, **k: ran.append(cmd))
    build.build_native()                      # no stamp
    build.build_native()                      # up to date
    assert len(ran) == 1 and f'-DRW4_TORCH_VERSION="{torch.__version__}"' in ran[0]
    monkeypatch.setattr(torch, "__version__", "9.9.9")
    build.build_native()
    build.build_native()
    assert len(ran) == 2


def test_it_is_not_used_beside_another_torch():
    assert kernels._native.torch_version == torch.__version__
    p = python("import warnings; warnings.simplefilter('error', DeprecationWarning)\n"
               "import torch; torch.__version__ = '9.9.9'\n"
               "from rocketllm_b200 import kernels\n"
               "print(kernels._native)")
    assert p.returncode == 0, p.stderr
    assert p.stdout.split()[-1] == "None" and "built against torch" in p.stderr
