"""The build recompiles what its sources, headers, or its own flags have changed since; with a compiler that only writes
down what it was asked."""
import importlib
import os
import stat
import sys

import pytest

STUB = """#!{python}
import sys
args = sys.argv[1:]
open(args[args.index("-o") + 1], "w").write("built")
open({log!r}, "a").write(" ".join(args) + "\\n")
"""


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """A build of two sources in a folder of its own; asked() gives what was compiled or linked since it was last called."""
    build = importlib.import_module("pir_amd.build")
    log, compiler = str(tmp_path / "log"), tmp_path / "compiler"
    compiler.write_text(STUB.format(python=sys.executable, log=log))
    compiler.chmod(compiler.stat().st_mode | stat.S_IXUSR)
    src = tmp_path / "csrc"
    src.mkdir()
    (tmp_path / "include").mkdir()
    for name in ("a.hip", "b.hip", "common.h", "optim_host.cpp"):
        (src / name).write_text("")
    (tmp_path / "pkg").mkdir()
    (tmp_path / "include" / "pir_hip.h").write_text("")
    (tmp_path / "build.py").write_text("")
    for k, v in dict(HERE=str(tmp_path / "pkg"), CSRC=str(src), OUT=str(tmp_path / "lib.so"), SOURCES=["a.hip", "b.hip"],
                     HOST_SRC=str(src / "optim_host.cpp"), HOST_OUT=str(tmp_path / "host.so"),
                     __file__=str(tmp_path / "build.py")).items():
        monkeypatch.setattr(build, k, v)
    monkeypatch.setenv("HIPCC", str(compiler))
    monkeypatch.setenv("CXX", str(compiler))
    for folder, _, files in os.walk(tmp_path):
        for f in files:
            os.utime(os.path.join(folder, f), (1e9, 1e9))

    def asked():
        lines = open(log).read().splitlines() if os.path.exists(log) else []
        if lines:
            os.remove(log)
        return sorted(os.path.basename(x.split(" -o ")[1].split()[0]) for x in lines)
    return tmp_path, build, asked


def test_nothing_is_compiled_twice(tree):
    _, build, asked = tree
    build.build(verbose=False)
    assert asked() == ["a.o", "b.o", "host.so", "lib.so"]
    build.build(verbose=False)
    assert asked() == []
    build.build(force=True, verbose=False)
    assert asked() == ["a.o", "b.o", "host.so", "lib.so"]


@pytest.mark.parametrize("changed, compiled", [
    ("csrc/a.hip", ["a.o", "lib.so"]), ("csrc/common.h", ["a.o", "b.o", "lib.so"]), ("csrc/optim_host.cpp", ["host.so"]),
    ("include/pir_hip.h", ["a.o", "b.o", "host.so", "lib.so"]),
    ("build.py", ["a.o", "b.o", "host.so", "lib.so"]),   # the flags stand there
])
def test_what_changed_is_compiled(tree, changed, compiled):
    root, build, asked = tree
    build.build(verbose=False)
    asked()
    new = os.path.getmtime(build.OUT) + 10
    os.utime(root / changed, (new, new))
    build.build(verbose=False)
    assert asked() == compiled


def test_the_entry_point_compiles_every_time(tree, monkeypatch):
    """Also where everything is built and up to date."""
    import __graft_entry__
    from pir_amd import _lib, optim
    _, build, asked = tree
    monkeypatch.setattr(_lib, "lib", lambda: None)
    monkeypatch.setattr(optim, "_host", lambda: None)
    for _ in range(2):
        __graft_entry__.build()
        assert asked() == ["a.o", "b.o", "host.so", "lib.so"]
