"""What `make lib` builds with and without torch."""

from __future__ import annotations

import os
import subprocess
import sys

from tests.common import ROOT


def _make(python):
    """The commands of `make lib` where the binding's source is newer than the binding."""
    r = subprocess.run(["make", "-n", "-W", "flashgann_b200/csrc/fg_torch.cpp", "lib", f"PYTHON={python}"], cwd=ROOT,
                       capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    return r.stdout


def test_the_library_builds_without_torch(tmp_path):
    """Where python has no torch (or there is none) the library is built and the binding is left out with a message."""
    bare = tmp_path / "python"  # an interpreter that sees no installed packages
    bare.write_text(f"#!/bin/sh\nexec {sys.executable} -S \"$@\"\n")
    os.chmod(bare, 0o755)
    for python in (str(bare), str(tmp_path / "none")):
        out = _make(python)
        assert "fg_torch.cpp" not in out and "no torch with CUDA" in out


def test_the_binding_is_built_with_torch():
    assert "csrc/fg_torch.cpp -o flashgann_b200/_torch_ops.so" in _make(sys.executable)


def test_star_import_needs_no_torch():
    """The search without torch: a plain and a star import work, and a call that needs it says so."""
    code = ("import sys\nsys.modules['torch'] = None\nfrom flashgann_b200 import *\nimport flashgann_b200 as fg\n"
            "lib(); compute_recall; search_multi\n"
            "try:\n    fg.kv_plan\nexcept ImportError as e:\n    print('needs', e.name)\n")
    r = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    assert r.stdout == "needs torch\n"


def test_cache_and_attention_calls_load_on_first_use():
    import flashgann_b200 as fg
    for name in ("KVPlan", "kv_plan", "kv_append", "paged_attention", "retrieved_attention"):
        assert callable(getattr(fg, name))
