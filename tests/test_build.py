"""What the build asks for, and when it builds again."""
import os
import stat
import sys
import sysconfig

import pytest

from darknet_b200 import build


@pytest.fixture
def elsewhere(tmp_path, monkeypatch):
    """Outputs under tmp_path, and an nvcc that writes an empty file where it is told to."""
    nvcc = tmp_path / "bin" / "nvcc"
    nvcc.parent.mkdir()
    nvcc.write_text('#!/bin/sh\nwhile [ "$1" != -o ]; do shift; done\n: > "$2"\n')
    nvcc.chmod(nvcc.stat().st_mode | stat.S_IXUSR)
    monkeypatch.setenv("NVCC", str(nvcc))
    monkeypatch.setattr(build, "PKG_DIR", str(tmp_path))
    monkeypatch.setattr(build, "LIB_PATH", str(tmp_path / "libxnor_b200.so"))
    monkeypatch.setattr(build, "BINDING_PATH", str(tmp_path / "_fourbit.so"))
    return tmp_path


def test_the_library_is_built_without_torch(elsewhere, monkeypatch, capfd):
    monkeypatch.setitem(sys.modules, "torch", None)
    for force in (True, False):
        assert build.build(force=force) == build.LIB_PATH and os.path.exists(build.LIB_PATH)
    assert not os.path.exists(build.BINDING_PATH)
    assert "_fourbit.so" in capfd.readouterr().err


def test_the_library_is_built_without_pythons_headers(elsewhere, monkeypatch):
    pytest.importorskip("torch")
    paths = sysconfig.get_paths()
    monkeypatch.setattr(sysconfig, "get_paths", lambda: {**paths, "include": str(elsewhere)})
    assert os.path.exists(build.build(force=True)) and not os.path.exists(build.BINDING_PATH)


def test_a_binding_that_does_not_compile_leaves_the_library_built(elsewhere, monkeypatch):
    pytest.importorskip("torch")
    monkeypatch.setattr(build, "BINDINGS", str(elsewhere))          # (no source there)
    with pytest.raises(RuntimeError, match="is built; its binding"):
        build.build(force=True)
    assert os.path.exists(build.LIB_PATH) and not os.path.exists(build.BINDING_PATH)


def test_the_binding_is_built_again_for_another_torch(elsewhere, monkeypatch):
    torch = pytest.importorskip("torch")
    with open(build.BINDING_PATH, "wb") as fh:
        fh.write(f"..built for torch {torch.__version__};..".encode())
    assert not build._binding_stale(torch)
    monkeypatch.setattr(torch, "__version__", torch.__version__ + "1")
    assert build._binding_stale(torch)


def test_a_binding_for_another_torch_is_refused(monkeypatch):
    torch = pytest.importorskip("torch")
    from darknet_b200 import fourbit
    build.build()
    from darknet_b200 import _fourbit
    assert _fourbit.built_for == torch.__version__
    monkeypatch.setattr(torch, "__version__", "1.0")
    with pytest.raises(FileNotFoundError, match="built for torch"):
        fourbit._Calls().product
