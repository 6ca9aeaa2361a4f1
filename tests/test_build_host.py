"""The build's parts that need no GPU and compile nothing."""
import sys

import pytest

from rusty_engine_b200 import build


@pytest.mark.parametrize("missing", ["torch", "g++", "cuda"])
def test_the_c_library_builds_without_what_the_torch_entry_needs(monkeypatch, tmp_path, capsys, missing):
    """librmoe.so is for callers without torch too: where torch, its CUDA libraries or g++ are
    missing, the torch-tensor entry is left out, with a note."""
    monkeypatch.setattr(build, "BINDING", str(tmp_path / "_kv_ops.so"))
    if missing == "torch":
        monkeypatch.setitem(sys.modules, "torch", None)
    elif missing == "g++":
        monkeypatch.setenv("PATH", str(tmp_path))
    else:
        import torch

        monkeypatch.setattr(torch, "__file__", str(tmp_path / "torch" / "__init__.py"))
    assert build.build_binding() is None
    assert "_kv_ops.so not built" in capsys.readouterr().err
