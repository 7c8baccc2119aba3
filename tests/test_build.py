"""What the build makes where parts of the machine are missing or have changed.  Runs without a GPU."""
import sys

import pytest

from codecoder_b200 import _lib, build


@pytest.fixture
def elsewhere(monkeypatch, tmp_path):
    """build() with the outputs in tmp_path and the compilers replaced by notes of their calls."""
    calls = []

    def write(name):
        def f(*a, **k):
            calls.append(name)
            (tmp_path / name).write_text("built")
            return str(tmp_path / name)
        return f
    monkeypatch.setattr(build, "OUT", str(tmp_path / "libbpc.so"))
    monkeypatch.setattr(build, "TORCH_OUT", str(tmp_path / "_torch_ops.so"))
    monkeypatch.setattr(build, "build_lib", write("libbpc.so"))
    return calls, write, tmp_path


def test_the_c_library_builds_without_torch(elsewhere, monkeypatch, capsys):
    calls, _, tmp_path = elsewhere
    monkeypatch.setitem(sys.modules, "torch", None)             # `import torch` raises ImportError
    assert build.build() == str(tmp_path / "libbpc.so") and calls == ["libbpc.so"]
    assert "torch cannot be imported" in capsys.readouterr().err
    assert not (tmp_path / "_torch_ops.so").exists()
    assert build.build(force=True) and calls == ["libbpc.so"] * 2


def test_the_c_library_builds_without_torchs_headers(elsewhere, monkeypatch, capsys):
    import torch
    calls, _, tmp_path = elsewhere
    monkeypatch.setattr(torch, "__file__", str(tmp_path / "torch" / "__init__.py"))
    assert build.build() and calls == ["libbpc.so"]
    assert "CUDAGuard.h is missing" in capsys.readouterr().err


def test_a_compiler_error_is_raised(elsewhere, monkeypatch):
    def fails():
        raise RuntimeError("g++ on torch_ops.cpp failed")
    monkeypatch.setattr(build, "build_torch_ops", fails)
    with pytest.raises(RuntimeError, match="g\\+\\+"):
        build.build()


def test_the_torch_side_says_that_it_is_missing(monkeypatch, tmp_path):
    monkeypatch.setattr(_lib, "_torch", None)
    monkeypatch.setattr(_lib, "_PKG", str(tmp_path))
    with pytest.raises(RuntimeError, match="missing.*headers"):
        _lib.torch_ops()
