"""The build's order: libmpl.so does not wait for what the extension module needs."""

import os

import pytest

from model_amd import build


@pytest.mark.parametrize("error", [ImportError("No module named 'torch'"), RuntimeError("g++ failed")])
def test_library_is_linked_without_the_extension(monkeypatch, tmp_path, error):
    linked = []

    def fails():
        raise error

    monkeypatch.setattr(build, "OBJ", str(tmp_path))
    monkeypatch.setattr(build, "_compile", lambda src, cc: src + ".o")
    monkeypatch.setattr(build, "_compile_ops", fails)
    monkeypatch.setattr(build, "_link", lambda cmd, out: linked.append(os.path.basename(out)))
    with pytest.raises(RuntimeError, match="libmpl.so is built.*_ops.so is not") as e:
        build.build()
    assert str(error) in str(e.value) and linked == ["libmpl.so"]


def test_both_are_linked(monkeypatch, tmp_path):
    linked = []
    monkeypatch.setattr(build, "OBJ", str(tmp_path))
    monkeypatch.setattr(build, "_compile", lambda src, cc: src + ".o")
    monkeypatch.setattr(build, "_compile_ops", lambda: "ops.o")
    monkeypatch.setattr(build, "_link", lambda cmd, out: linked.append(os.path.basename(out)))
    assert build.build() == build.LIB and linked == ["libmpl.so", "_ops.so"]
