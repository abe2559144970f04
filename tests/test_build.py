"""CPU checks of build_lib's order: the library needs hipcc alone, and never
stands beside an extension of another build."""

import os

import pytest

import conftest  # noqa: F401  (paths)
import build_lib


@pytest.fixture
def built(tmp_path, monkeypatch):
    """Paths of an earlier build's library and extension, and a compiler that
    fails for the sources named in `failing`."""
    lib, ext = str(tmp_path / "lib.so"), str(tmp_path / "ext.so")
    failing = set()

    def run(cmd, verbose):
        for f in failing:
            if any(os.path.basename(c) == f for c in cmd):
                raise RuntimeError(f"{f} does not compile")
        with open(cmd[cmd.index("-o") + 1], "w") as out:
            out.write("new")

    monkeypatch.setattr(build_lib, "_run", run)
    monkeypatch.setattr(build_lib, "OUT", lib)
    monkeypatch.setattr(build_lib, "EXT_OUT", ext)
    for p in (lib, ext):
        with open(p, "w") as f:
            f.write("old")
    return lib, ext, failing


def read(path):
    with open(path) as f:
        return f.read()


def test_both_are_built(built):
    lib, ext, _ = built
    assert build_lib.build(out=lib) == lib
    assert read(lib) == read(ext) == "new"


def test_the_library_is_built_without_the_extension(built):
    lib, ext, failing = built
    failing.add(build_lib.EXT_SOURCE)
    with pytest.warns(UserWarning, match="8-bit cache's calls are not built: kv8_bind.cpp"):
        build_lib.build(out=lib)
    assert read(lib) == "new" and not os.path.exists(ext)


def test_a_library_that_does_not_compile_leaves_both_as_they_were(built):
    lib, ext, failing = built
    failing.add("norm.hip")
    with pytest.raises(RuntimeError, match="norm.hip"):
        build_lib.build(out=lib)
    assert read(lib) == read(ext) == "old"


def test_the_host_compiler_is_the_users(monkeypatch):
    monkeypatch.setenv("CXX", "ccache some-c++")
    assert build_lib.host_cxx() == ["ccache", "some-c++"]
    monkeypatch.delenv("CXX")
    assert len(build_lib.host_cxx()) == 1
