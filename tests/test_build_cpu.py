"""What is built, for which interpreter, and what does not need what."""
import importlib.machinery
import re
from pathlib import Path

import pytest
import torch

from ghost_flow_b200.csrc import build as b
from ghost_flow_b200.ops import _lib


def test_the_module_is_this_interpreters():
    suffix = importlib.machinery.EXTENSION_SUFFIXES[0]
    path = Path(_lib.calls().__file__)
    assert path.name == "_gf_calls" + suffix and suffix.count(".") == 2 and path.parent == b.LIB_DIR


def test_the_declared_pytorch_has_the_interface_that_operators_go_through():
    need = re.search(r'"torch>=([\d.]+)"', (Path(b.__file__).parents[2] / "pyproject.toml").read_text()).group(1)
    assert (2, 11) <= tuple(map(int, need.split("."))) <= tuple(map(int, torch.__version__.split(".")[:2]))
    assert hasattr(torch.Tensor, "__dlpack_c_exchange_api__")


def test_the_libraries_are_linked_where_the_module_cannot_be_compiled(tmp_path, monkeypatch):
    for name, text in (("host.cpp", 'extern "C" int two() { return 2; }'), ("module.cpp", "#include <no_such_header_of_python.h>\n")):
        (tmp_path / name).write_text(text)
    for name, value in dict(HERE=tmp_path, OBJ_DIR=tmp_path / "build", LIB_DIR=tmp_path / "lib", CUDA_SOURCES=[], HOST_SOURCES=["host.cpp"],
                            PYTHON_SOURCES=["module.cpp"]).items():
        monkeypatch.setattr(b, name, value)
    with pytest.raises(RuntimeError, match="module.cpp"):
        b.build(checked=False)
    assert (tmp_path / "lib" / "libghostflow.so").exists() and not (tmp_path / "lib" / b.CALLS_NAME).exists()
    (tmp_path / "host.cpp").write_text("no c++")
    with pytest.raises(RuntimeError, match="host.cpp"):
        b.build(checked=False)
