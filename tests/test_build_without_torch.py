"""CPU: the C and C++ libraries build on a host without PyTorch; what is built on PyTorch is left out, and said to be."""
import importlib
import os
import sys

import __graft_entry__ as entry


def test_build_without_torch(pkg, monkeypatch, capsys):
    builder = importlib.import_module(entry.PKG_NAME + ".build")
    done = []
    monkeypatch.setattr(builder, "build_library", lambda *a: done.append("library"))
    monkeypatch.setattr(builder, "build_compat", lambda *a: done.append("compat"))
    monkeypatch.setitem(sys.modules, "torch", None)            # as if it were not installed
    binding = os.path.join(builder.HERE, "_q8.so")
    before = os.path.getmtime(binding) if os.path.exists(binding) else None
    assert builder.build(force=True) == builder.OUT
    assert done == ["library", "compat"] and "_q8.so" in capsys.readouterr().err
    assert (os.path.getmtime(binding) if os.path.exists(binding) else None) == before
