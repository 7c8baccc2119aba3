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


def test_another_torch_gets_another_build(elsewhere, monkeypatch):
    calls, write, tmp_path = elsewhere
    out = tmp_path / "_torch_ops.so"

    def compile_():
        calls.append("_torch_ops.so")
        out.write_bytes(b"code" + build.STAMP + build.torch_stamp().encode() + b"]more code")
    monkeypatch.setattr(build, "build_torch_ops", compile_)
    build.build()
    build.build()
    assert sorted(calls) == ["_torch_ops.so", "libbpc.so"]      # the second call found both in order
    import torch
    monkeypatch.setattr(torch, "__version__", "9.9.9")
    build.build()
    assert calls.count("_torch_ops.so") == 2 and "torch 9.9.9" in build.stamp_of(str(out))
    build.build()
    assert calls.count("_torch_ops.so") == 2
    out.write_bytes(b"a module from before the stamp")
    build.build()
    assert calls.count("_torch_ops.so") == 3


def test_the_built_module_is_refused_under_another_torch(monkeypatch):
    import torch
    build.build()
    assert build.stamp_of(build.TORCH_OUT) == build.torch_stamp()
    monkeypatch.setattr(_lib, "_torch", None)
    monkeypatch.setattr(torch, "__version__", "9.9.9")
    with pytest.raises(RuntimeError, match="built for torch .*9.9.9"):
        _lib.torch_ops()
