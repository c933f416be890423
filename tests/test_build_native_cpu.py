"""The build: the engine library needs nvcc alone, and the torch extension is for one torch and one interpreter."""

import os
import sys

import pytest

from forgetune_b200 import _native, build_native
from forgetune_b200.errors import ForgeTuneRuntimeError


@pytest.fixture
def elsewhere(monkeypatch, tmp_path):
    """The extension goes to a folder of the test, where there is none yet; the library counts as built."""
    newer = build_native._newer
    monkeypatch.setattr(build_native, "_newer", lambda t, files: t == build_native.LIB_PATH or newer(t, files))
    path = str(tmp_path / "_torch_ops.so")
    monkeypatch.setattr(build_native, "TORCH_OPS_PATH", path)
    return path


def fake_compiler(tmp_path, text):
    """A host compiler that notes its arguments and writes `text` as its output."""
    path = tmp_path / "fake-c++"
    path.write_text("#!%s\nimport sys\nopen(%r, 'a').write(' '.join(sys.argv[1:]) + '\\n')\n"
                    "open(sys.argv[sys.argv.index('-o') + 1], 'wb').write(%r)\n"
                    % (sys.executable, str(tmp_path / "ran"), text.encode()))
    path.chmod(0o755)
    return str(path)


def test_the_library_alone_where_the_extension_cannot_be_built(elsewhere, monkeypatch, tmp_path):
    real = build_native.sysconfig.get_paths
    monkeypatch.setattr(build_native.sysconfig, "get_paths", lambda *a, **k: dict(real(*a, **k), include=str(tmp_path)))
    with pytest.warns(UserWarning, match="Python.h"):
        assert build_native.build() == build_native.LIB_PATH
    assert not os.path.exists(elsewhere) and build_native.up_to_date()
    monkeypatch.setattr(_native, "_ops", None)
    with pytest.raises(ForgeTuneRuntimeError, match="not built"):
        _native.torch_ops()


def test_the_extension_takes_the_compiler_of_the_environment(elsewhere, monkeypatch, tmp_path):
    target = build_native.torch_ops_target()
    monkeypatch.setenv("CXX", fake_compiler(tmp_path, "_torch_ops built for: %s\0" % target))
    assert not build_native.up_to_date()
    build_native.build()
    ran = (tmp_path / "ran").read_text()
    assert "torch_ops.cpp" in ran and target in ran
    assert build_native.up_to_date()


@pytest.mark.parametrize("text", ["_torch_ops built for: torch 1.0 abc, cpython-27\0", "an extension without the line"])
def test_an_extension_for_another_torch_is_built_again_and_not_loaded(elsewhere, monkeypatch, tmp_path, text):
    monkeypatch.setenv("CXX", fake_compiler(tmp_path, text))
    build_native.build()
    assert not build_native.up_to_date()
    build_native.build()
    assert (tmp_path / "ran").read_text().count("torch_ops.cpp") == 2
    monkeypatch.setattr(_native, "_ops", None)
    with pytest.raises(ForgeTuneRuntimeError, match="is built for"):
        _native.torch_ops()


def test_the_extension_in_the_tree_is_for_this_torch():
    import sysconfig

    import torch
    built_for = build_native.torch_ops_built_for(build_native.TORCH_OPS_PATH)
    assert built_for == build_native.torch_ops_target()
    for part in (str(torch.__version__), torch.version.git_version, sysconfig.get_config_var("SOABI")):
        assert part in built_for


def test_a_compiler_with_arguments_and_one_that_is_not_there(elsewhere, monkeypatch, tmp_path):
    target = build_native.torch_ops_target()
    cxx = fake_compiler(tmp_path, "_torch_ops built for: %s\0" % target)
    monkeypatch.setenv("CXX", cxx + " -march=native")
    build_native.build()
    assert (tmp_path / "ran").read_text().startswith("-march=native ") and build_native.up_to_date()
    monkeypatch.setenv("CXX", str(tmp_path / "nowhere"))
    with pytest.raises(RuntimeError, match="nowhere"):
        build_native._build_torch_ops(False)


def test_no_nvcc_and_the_library_in_place(elsewhere, monkeypatch):
    monkeypatch.delenv("NVCC", raising=False)
    monkeypatch.setattr(build_native, "nvcc", lambda: (_ for _ in ()).throw(RuntimeError("nvcc not found")))
    with pytest.warns(UserWarning, match="nvcc"):
        assert build_native.build() == build_native.LIB_PATH
