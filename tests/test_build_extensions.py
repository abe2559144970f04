"""CPU checks of the extension modules' build: each stands or is left out by
itself, and none of another build stays beside a new library."""

import os

import pytest

import conftest  # noqa: F401  (paths)
import build_lib


@pytest.fixture
def built(tmp_path, monkeypatch):
    """An earlier build's files, and a compiler that fails for the sources in
    `failing`."""
    lib = str(tmp_path / "lib.so")
    monkeypatch.setattr(build_lib, "OUT", lib)
    monkeypatch.setattr(build_lib, "EXT_OUT", str(tmp_path / "_kv8_ext.so"))
    paths = {source: path for source, path, _ in build_lib._extensions()}
    failing = set()

    def run(cmd, verbose):
        if any(os.path.basename(c) in failing for c in cmd):
            raise RuntimeError("does not compile")
        with open(cmd[cmd.index("-o") + 1], "w") as out:
            out.write("new")

    monkeypatch.setattr(build_lib, "_run", run)
    for p in (lib, *paths.values()):
        with open(p, "w") as f:
            f.write("old")
    return lib, paths, failing


def read(path):
    with open(path) as f:
        return f.read()


def test_all_are_built(built):
    lib, paths, _ = built
    assert set(paths) == {"kv8_bind.cpp", "gen_bind.cpp"} and len(set(paths.values())) == 2
    assert build_lib.build(out=lib) == lib
    assert read(lib) == "new" and all(read(p) == "new" for p in paths.values())
    assert sorted(build_lib.build_ext()) == sorted(paths.values())


@pytest.mark.parametrize("source,what", [("kv8_bind.cpp", "8-bit cache's calls"), ("gen_bind.cpp", "generation calls")])
def test_one_that_does_not_compile_is_left_out(built, source, what):
    lib, paths, failing = built
    failing.add(source)
    with pytest.warns(UserWarning, match=f"{what} are not built"):
        build_lib.build(out=lib)
    assert read(lib) == "new" and not os.path.exists(paths[source])
    assert all(read(p) == "new" for s, p in paths.items() if s != source)


def test_one_module_at_a_given_path(built, tmp_path):
    """build_ext(out=path): the 8-bit cache's module alone, there."""
    _, paths, _ = built
    to = str(tmp_path / "elsewhere.so")
    assert build_lib.build_ext(out=to) == to and build_lib.build_ext(False, to) == to
    assert read(to) == "new" and all(read(p) == "old" for p in paths.values())
