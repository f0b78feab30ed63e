"""CPU checks of the build: the library without torch, and when the torch
module has to be built anew."""
import importlib
import os
import sys

import pytest

from provenloop_b200 import adapters, build


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """A tree of one small source and a torch module that does not compile."""
    (tmp_path / "one.cu").write_text('extern "C" int one() { return 1; }\n')
    (tmp_path / "torch_ops.cpp").write_text("#error headers of another torch\n")
    for name, value in dict(CSRC=str(tmp_path), LIB=str(tmp_path / "lib.so"), TORCH_OPS=str(tmp_path / "ops.so"), SOURCES=["one.cu"],
                            HEADERS=[]).items():
        monkeypatch.setattr(build, name, value)
    return tmp_path


def test_library_without_torch(tree, monkeypatch, capsys):
    monkeypatch.setattr(build, "have_torch", lambda: False)
    monkeypatch.setitem(sys.modules, "torch", None)  # importing it fails
    assert build.needs_build()
    assert build.build() == build.LIB and os.path.exists(build.LIB)
    assert "torch is not installed" in capsys.readouterr().err
    assert not build.needs_build()


@pytest.mark.parametrize("broken", ["headers", "import", "compiler"])
def test_library_beside_a_torch_that_does_not_build(tree, monkeypatch, broken):
    if broken == "import":
        monkeypatch.setattr(build, "torch_ops_command", lambda out: importlib.import_module("no_such_torch"))
    if broken == "compiler":
        monkeypatch.setattr(build, "torch_ops_command", lambda out: [str(tree / "no_such_compiler")])
    with pytest.raises(RuntimeError, match="torch_ops.cpp"):
        build.build()
    assert os.path.exists(build.LIB)
    assert build.needs_build()  # the module is still missing
    before = os.path.getmtime(build.LIB)
    with pytest.raises(RuntimeError, match="torch_ops.cpp"):
        build.build()
    assert os.path.getmtime(build.LIB) == before  # the library is not built again for it


def test_module_of_another_torch_is_stale(tree, monkeypatch):
    (tree / "lib.so").write_bytes(b"")
    (tree / "ops.so").write_bytes(b"..." + build.torch_tag().encode() + b"\0...")
    assert not build.needs_build()
    real = build.importlib.metadata.version
    monkeypatch.setattr(build.importlib.metadata, "version", lambda name: "0.1" if name == "torch" else real(name))
    assert build.needs_build() and build.torch_ops_stale()
    monkeypatch.setattr(adapters, "_ops", None)
    monkeypatch.setattr(adapters, "HERE", str(tree))
    (tree / "_torch_ops.so").write_bytes(b"")
    with pytest.raises(ImportError, match="torch 0.1"):
        adapters._load()


def test_module_says_what_it_is_for():
    assert adapters._load().built_for == build.torch_tag()
    assert build.torch_ops_fits()
