"""Which Python and which torch the compiled binding is for: its file's name, the check at
import, and the build's decision to make it again."""
import importlib.util
import os
import sysconfig

import pytest

from test_serving_cpu import _lib

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "atflash-kernel_b200")


@pytest.fixture
def build(tmp_path, monkeypatch):
    """build.py with its binding elsewhere and a compiler that only writes the file"""
    spec = importlib.util.spec_from_file_location("atflash_build_test", os.path.join(PKG, "build.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    m.runs = []

    def run(cmd, check):
        m.runs.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write("binding")

    monkeypatch.setattr(m.subprocess, "run", run)
    monkeypatch.setattr(m, "nvcc_path", lambda: "/usr/local/cuda/bin/nvcc")
    monkeypatch.setattr(m, "BINDING", str(tmp_path / os.path.basename(m.BINDING)))
    return m


def test_the_file_belongs_to_one_python(build, tmp_path):
    suffix = sysconfig.get_config_var("EXT_SUFFIX")
    assert "cpython" in suffix and os.path.basename(build.BINDING) == "_binding" + suffix
    (tmp_path / "_binding.so").write_text("any Python's")
    build.build_binding()
    assert os.path.exists(build.BINDING) and not (tmp_path / "_binding.so").exists()


def test_built_again_for_another_torch(build, monkeypatch):
    import torch
    build.build_binding()
    build.build_binding()
    assert len(build.runs) == 1
    with open(build.BINDING + ".torch") as f:
        assert f.read() == torch.__version__
    # an older torch, whose files are all older than the binding
    monkeypatch.setattr(build, "torch_version", lambda torch_dir: "1.0.0")
    build.build_binding()
    build.build_binding()
    assert len(build.runs) == 2
    os.remove(build.BINDING + ".torch")  # one whose torch nobody knows
    build.build_binding()
    assert len(build.runs) == 3
    build.build_binding(force=True)
    assert len(build.runs) == 4


def test_another_pythons_file_is_not_loaded(monkeypatch, tmp_path):
    ffi, _ = _lib()
    monkeypatch.setattr(ffi, "_bind", None)
    monkeypatch.setattr(ffi, "_BINDING_PATH", str(tmp_path / "_binding.cpython-39-x86_64-linux-gnu.so"))
    with pytest.raises(ImportError, match="not been built for this Python.*build it again"):
        ffi.binding()


def test_the_loaded_one_is_this_pythons():
    ffi, _ = _lib()
    if not os.path.exists(ffi._BINDING_PATH):
        pytest.skip("binding not built")
    assert ffi.binding().__file__ == ffi._BINDING_PATH
