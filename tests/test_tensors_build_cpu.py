"""The compiled looks at tensors: built when they are missing, old or another torch's, and used by the process that builds them."""
import os
import shutil
import subprocess
import sys

import pytest
import torch

from promptcache_amd import _blocks as B
from promptcache_amd import _buildlib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture
def place(tmp_path, monkeypatch):
    """A folder with sources and a blocks library that is newer than all of them."""
    src, pkg = tmp_path / "csrc", tmp_path / "pkg"
    src.mkdir(), pkg.mkdir()
    for f in (src / "pb_x.hip", src / "py_tensors.cpp"):
        f.write_text("")
        os.utime(f, (1000, 1000))
    lib = pkg / "libpromptcache_blocks.so"
    lib.write_text("")
    monkeypatch.setattr(_buildlib, "CSRC", str(src))
    monkeypatch.setattr(_buildlib, "PKG", str(pkg))
    monkeypatch.setattr(_buildlib, "INCLUDE", str(tmp_path))
    built = []

    def build():
        built.append(1)
        (pkg / "_tensors.so").write_text("")
    monkeypatch.setattr(_buildlib, "build_tensors", build)
    return src, pkg, built


def test_the_blocks_group_renews_what_is_missing_or_old(place):
    src, pkg, built = place
    _buildlib.build("blocks")
    assert len(built) == 1                                          # missing, beside a library that is up to date
    _buildlib.build("blocks")
    assert len(built) == 1
    os.utime(pkg / "_tensors.so", (999, 999))
    _buildlib.build("blocks")
    assert len(built) == 2                                          # older than its source
    _buildlib.build("blocks")
    assert len(built) == 2


def python(folder, code):
    """Runs a copy of the package in a process of its own; the build of the helper is replaced by a copy of the one that is there (``real``), and counted."""
    out = subprocess.run([sys.executable, "-c", f"import sys, shutil; sys.path.insert(0, {str(folder)!r})\nfrom promptcache_amd import _buildlib\nbuilt = []\n"
                          f"import os\ndef build():\n    built.append(1); new = _buildlib.tensors_path() + '.new'; shutil.copy({str(folder / 'real.so')!r}, new); os.replace(new, _buildlib.tensors_path())\n"
                          "_buildlib.build_tensors = build\n"
                          "import promptcache_amd._blocks as B\n" + code], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stderr
    return out.stdout.split()


@pytest.fixture
def copy(tmp_path):
    if not (os.path.exists(_buildlib.tensors_path()) and os.path.exists(B.lib_path())):
        pytest.skip("nothing is built here")
    pkg = tmp_path / "promptcache_amd"
    pkg.mkdir()
    (tmp_path / "csrc").mkdir()
    (pkg / "__init__.py").write_text("")
    for f in ("_blocks.py", "_buildlib.py"):
        shutil.copy(os.path.join(_buildlib.PKG, f), pkg / f)
    (pkg / "libpromptcache_blocks.so").symlink_to(B.lib_path())
    shutil.copy(_buildlib.tensors_path(), tmp_path / "real.so")
    return tmp_path, pkg


SHOW = "\nB.load(); t = sys.modules.get('promptcache_amd._tensors'); print(len(built), B._flat is getattr(t, 'flat', None), B._pool is getattr(t, 'pool', None))"


def test_a_process_that_finds_none_builds_and_uses_them(copy):
    folder, pkg = copy
    assert python(folder, SHOW) == ["1", "True", "True"]
    assert python(folder, SHOW) == ["0", "True", "True"]


def test_those_that_cannot_be_loaded_are_built_anew(copy):
    folder, pkg = copy
    (pkg / "_tensors.so").write_text("no library")
    assert python(folder, SHOW) == ["1", "True", "True"]


def test_another_torchs_serve_nobody_and_are_built_anew(copy):
    """The process that has loaded them already looks in Python."""
    folder, pkg = copy
    shutil.copy(folder / "real.so", pkg / "_tensors.so")
    assert python(folder, "import torch; B._compiled = False; B._flat, B._heads, B._table, B._pool = B._looks; torch.__version__ = '0.1'" + SHOW) == ["1", "False", "False"]
    assert python(folder, SHOW) == ["0", "True", "True"]


def test_none_are_built_where_nothing_is_to_be_built(copy):
    folder, pkg = copy
    assert python(folder, SHOW.replace("load()", "load(False)")) == ["0", "False", "False"]


def test_this_process_uses_them():
    if not os.path.exists(_buildlib.tensors_path()):
        pytest.skip("nothing is built here")
    B.load()
    from promptcache_amd import _tensors
    assert _tensors.torch_version == torch.__version__.split("+")[0] and B._flat is _tensors.flat
