"""The binding is a shortcut: a build for another PyTorch, or none, costs host time and nothing else."""
import os
import warnings

import pytest

import __graft_entry__ as entry
from dcnv4_b200 import _lib, build


@pytest.fixture(scope="module", autouse=True)
def built():
    entry.build()


def test_the_binding_is_found_by_its_pytorch(monkeypatch):
    import torch
    assert torch.__version__.split("+")[0] in os.path.basename(_lib.bindings_path())
    assert os.path.exists(_lib.bindings_path()) and build.is_current()
    monkeypatch.setattr(torch, "__version__", "1.0.0+other")
    assert not os.path.exists(_lib.bindings_path()) and not build.is_current()


@pytest.mark.parametrize("kind", ["missing", "not a library", "for another interface"])
def test_a_binding_that_cannot_be_used(kind, tmp_path, monkeypatch):
    path = tmp_path / "dcnv4_b200_bindings.so"
    if kind == "not a library":
        path.write_bytes(b"\x7fELF but no more")
    elif kind == "for another interface":
        monkeypatch.setattr(_lib.importlib.util, "module_from_spec", lambda spec: _Old)
        path = _lib.bindings_path()
    monkeypatch.setattr(_lib, "bindings_path", lambda: str(path))
    monkeypatch.setattr(_lib, "_bindings", None)
    with pytest.warns(RuntimeWarning, match="cannot be used"):
        got = _lib.bindings()
    assert got.ln_forward(0, None) is None and got.ln_backward(1) is None
    with warnings.catch_warnings():                       # once
        warnings.simplefilter("error")
        assert _lib.bindings() is got


class _Old:
    @staticmethod
    def init(a, b, c):
        raise AssertionError("unreachable: four addresses are handed over")
