"""What the in-tree build takes for up to date (no GPU, no compiler run)."""

import glob
import os
import shutil
import sys

import pytest

from wanferenz_b200 import _build
from wanferenz_b200 import _lib as L


def test_every_source_and_header_of_the_library_is_watched():
    """Headers with inline code count, whatever their suffix: an edit of one alone makes the library stale."""
    here = {os.path.join(_build.CSRC, f) for f in os.listdir(_build.CSRC)}
    device = {f for f in here if f.endswith((".cu", ".cuh", ".h"))}
    assert device and device <= set(_build.deps())
    assert set(glob.glob(os.path.join(_build.ROOT, "include", "*.h"))) <= set(_build.deps())


@pytest.fixture
def entry(tmp_path, monkeypatch):
    """A Python entry module of the present source, torch and interpreter, in a folder of its own."""
    L.load_ext()
    for name in ("EXT", "EXT_KEY"):
        shutil.copy(getattr(_build, name), tmp_path)
        monkeypatch.setattr(_build, name, str(tmp_path / os.path.basename(getattr(_build, name))))
    src = tmp_path / "wf_torch.cpp"
    shutil.copy(_build.EXT_SRC, src)
    monkeypatch.setattr(_build, "EXT_SRC", str(src))
    monkeypatch.setattr(L, "_EXT", None)
    return src


def test_the_entry_module_in_place_is_current(entry):
    assert _build.ext_current() and _build.build_ext() == _build.EXT


@pytest.mark.parametrize("what", ["torch", "source", "key", "module"])
def test_a_stale_entry_module_is_not_loaded(entry, monkeypatch, what):
    """One built for another torch or from another source would be called with arguments that it does not have."""
    if what == "torch":
        monkeypatch.setattr("torch.__version__", "1.0.0")
    elif what == "source":
        entry.write_text(entry.read_text() + "// another\n")
    else:
        os.remove(_build.EXT if what == "module" else _build.EXT_KEY)
    assert not _build.ext_current()
    with pytest.raises(ImportError, match="entry module"):
        L.load_ext(build_if_missing=False)


@pytest.mark.parametrize("lacks", ["compiler", "headers", "torch"])
def test_the_library_builds_without_what_the_entry_module_needs(monkeypatch, capsys, lacks):
    """A host of the C ABI has nvcc; the command builds the library there, says what is left out, and succeeds."""
    monkeypatch.setattr(_build, "build", lambda force=False, verbose=False: "the library")
    if lacks == "compiler":
        monkeypatch.setenv("CXX", "/nonexistent/g++")
    elif lacks == "headers":
        monkeypatch.setattr("sysconfig.get_paths", lambda: {"include": "/nonexistent"})
    else:
        monkeypatch.setitem(sys.modules, "torch", None)
    _build.main(["_build", "--force"])
    seen = capsys.readouterr()
    assert "the library" in seen.out and "not built" in seen.err


def test_an_entry_module_that_does_not_compile_is_an_error(entry, monkeypatch):
    monkeypatch.setattr(_build, "build", lambda force=False, verbose=False: "the library")
    entry.write_text("#error no\n")
    with pytest.raises(RuntimeError, match="failed"):
        _build.main(["_build"])


def test_a_package_without_its_sources_loads_the_module_it_came_with(entry, monkeypatch):
    """Copied with its built libraries alone: torch and Python still have to be those it was built for."""
    os.remove(entry)
    assert _build.ext_current()
    assert L.load_ext(build_if_missing=False)
    monkeypatch.setattr("torch.__version__", "1.0.0")
    assert not _build.ext_current()
