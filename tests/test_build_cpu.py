"""The library and the torch binding are built and loaded one without the other, in a copy of the
package."""

import os
import shutil
import subprocess
import sys

import pytest

from conftest import ROOT

PACKAGE = "cs348k_fast_attention_grammar_b200"


@pytest.fixture
def tree(tmp_path):
    """A copy of the package and its header whose library is fresh and whose binding is missing."""
    def skip(folder, names):
        return [n for n in names if n.startswith(("_fa_torch", "__pycache__")) or n.endswith(".lock")]

    shutil.copytree(os.path.join(ROOT, PACKAGE), tmp_path / PACKAGE, ignore=skip)
    shutil.copytree(os.path.join(ROOT, "include"), tmp_path / "include")
    library = tmp_path / PACKAGE / "libfa_b200.so"
    if not library.exists():
        pytest.skip("the library is not built")
    os.utime(library)
    return tmp_path


def _run(tree, code, **env):
    code = f"from {PACKAGE} import _lib, build\n" + code
    return subprocess.run([sys.executable, "-c", code], cwd=tree, env={**os.environ, **env},
                          capture_output=True, text=True, timeout=300)


def _left_over(tree):
    return [p.name for p in (tree / PACKAGE).iterdir() if p.suffix == ".tmp"]


def test_the_library_loads_without_the_binding(tree):
    r = _run(tree, "assert _lib.load().fa_version() > 0\n"
                   "try:\n"
                   "    _lib.load_binding()\n"
                   "except RuntimeError as e:\n"
                   "    print('no binding:', e)\n"
                   "assert _lib.load().fa_version() > 0\n", CXX="false")
    assert r.returncode == 0 and "no binding: false failed" in r.stdout, r.stdout + r.stderr
    assert not _left_over(tree)


def test_the_binding_builds_when_it_is_asked_for(tree):
    r = _run(tree, "assert build.binding_stale() and not build.library_stale()\n"
                   "m = _lib.load_binding()\n"
                   "assert m is _lib.load_binding() and not build.is_stale()\n"
                   "print(m.__name__)\n")
    assert r.returncode == 0 and "_fa_torch" in r.stdout, r.stdout + r.stderr


def test_a_missing_compiler_leaves_no_other_behind(tree):
    """One compiler that cannot be started: the other ends its work, and nothing is left over."""
    fake = tree / "nvcc"
    fake.write_text("#!/bin/sh\nsleep 1\nwhile [ \"$1\" != -o ]; do shift; done\necho made > \"$2\"\n")
    fake.chmod(0o755)
    r = _run(tree, "try:\n"
                   "    build.build(force=True)\n"
                   "except RuntimeError as e:\n"
                   "    print('failed:', e)\n", NVCC=str(fake), CXX=str(tree / "none" / "g++"))
    assert r.returncode == 0 and "failed: g++" in r.stdout, r.stdout + r.stderr
    assert (tree / PACKAGE / "libfa_b200.so").read_text() == "made\n"
    assert not _left_over(tree)


def test_a_binding_of_another_torch_is_stale(tree):
    """The binding reads torch's objects through inlined code: one that another torch or Python
    built is not loaded."""
    for built in (p for p in os.listdir(os.path.join(ROOT, PACKAGE)) if p.startswith("_fa_torch")):
        shutil.copy(os.path.join(ROOT, PACKAGE, built), tree / PACKAGE)      # (for its time)
    r = _run(tree, "import torch\n"
                   "_lib.load_binding()\n"
                   "assert not build.binding_stale()\n"
                   "mine, torch.__version__ = torch.__version__, '0.0.1'\n"
                   "assert build.binding_stale()\n"
                   "torch.__version__ = mine\n"
                   "assert not build.binding_stale()\n"
                   "import sysconfig\n"
                   "sysconfig.get_config_vars()['SOABI'] = 'other'\n"
                   "assert build.binding_stale()\n")
    assert r.returncode == 0, r.stdout + r.stderr
