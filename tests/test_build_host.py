"""The build recipe with stand-ins for the compilers: the library does not wait for the host binding."""
import os
import sys

import pytest

from ragrt_b200 import build as B

COMPILER = """#!/bin/sh
echo run >> {log}
while [ $# -gt 0 ]; do
    if [ "$1" = -o ]; then echo made > "$2"; fi
    shift
done
exit {status}
"""


def compiler(path, status=0):
    path.write_text(COMPILER.format(log=f"{path}.log", status=status))
    path.chmod(0o755)
    return str(path)


def runs(path):
    return len(open(f"{path}.log").read().split()) if os.path.exists(f"{path}.log") else 0


@pytest.fixture
def tree(tmp_path, monkeypatch):
    monkeypatch.setattr(B, "OBJ_DIR", str(tmp_path / "obj"))
    monkeypatch.setattr(B, "LIB", str(tmp_path / "lib.so"))
    monkeypatch.setattr(B, "BIND", str(tmp_path / "bind.so"))
    monkeypatch.setattr(B, "NVCC", compiler(tmp_path / "nvcc"))
    monkeypatch.setattr(B, "CXX", compiler(tmp_path / "cxx"))
    return tmp_path


def test_library_and_binding_are_built_once(tree):
    B.build()
    assert os.path.exists(B.LIB) and os.path.exists(B.BIND) and runs(B.CXX) == 1
    n = runs(B.NVCC)
    assert n == len(B._sources()) + 1
    B.build()
    assert runs(B.NVCC) == n and runs(B.CXX) == 1


@pytest.mark.parametrize("why", ["fails", "missing", "no torch"])
def test_library_without_a_binding(tree, monkeypatch, capsys, why):
    open(B.BIND, "w").write("of an earlier interface")
    if why == "fails":
        B.CXX = compiler(tree / "bad", 1)
    elif why == "missing":
        B.CXX = str(tree / "nowhere")
    else:
        monkeypatch.setitem(sys.modules, "torch", None)
    assert B.build() == B.LIB
    assert os.path.exists(B.LIB) and not os.path.exists(B.BIND)
    assert "without its host binding" in capsys.readouterr().err


def test_a_kernel_that_does_not_compile_is_an_error(tree):
    B.NVCC = compiler(tree / "bad", 1)
    with pytest.raises(RuntimeError, match="nvcc failed"):
        B.build()
    assert not os.path.exists(B.LIB)
