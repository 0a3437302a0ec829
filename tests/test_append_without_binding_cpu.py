"""The append where the compiled binding is missing: it goes on over ctypes, says so, and
refuses what it refuses otherwise."""
import pytest
import torch

from test_serving_cpu import _lib


@pytest.fixture
def no_binding(monkeypatch, tmp_path):
    ffi, _ = _lib()
    monkeypatch.setattr(ffi, "_bind", None)
    monkeypatch.setattr(ffi, "_BINDING_PATH", str(tmp_path / "none.so"))
    return ffi


def test_the_append_gets_past_the_missing_binding(no_binding):
    import atflash
    i, x = torch.zeros(1, dtype=torch.int32), torch.zeros((1, 1, 128), dtype=torch.bfloat16)
    s = torch.ones((1, 1))
    with pytest.warns(RuntimeWarning, match="ctypes"), pytest.raises(ValueError, match="CUDA"):
        atflash.append_paged_kv_cache(x, x, i, i, (x[None], x[None]), i, i)
    with pytest.warns(RuntimeWarning, match="ctypes"), pytest.raises(ValueError, match="CUDA"):
        atflash.append_paged_kv_cache(x, x, i, i, (x[None], x[None]), i, i, kv_scales=(s, s))


def test_what_needs_the_binding_says_so(no_binding):
    import atflash
    i, x = torch.zeros(1, dtype=torch.int32), torch.zeros((1, 1, 128), dtype=torch.bfloat16)
    w, c = torch.ones(128), torch.zeros((2, 64))
    with pytest.raises(ImportError, match="build it again"):
        atflash.append_paged_kv_cache(x, x, i, i, (x[None], x[None]), i, i, rope=(c, c), k_norm=(w, 1e-6))
    with pytest.raises(ImportError, match="build it again"):
        atflash.qk_norm_rope(x, None, w, None, c, c)


def test_a_missing_library_is_said_without_a_detour(monkeypatch, tmp_path):
    import warnings

    import atflash
    ffi, _ = _lib()
    monkeypatch.setattr(ffi, "_bind", None)
    monkeypatch.setattr(ffi, "_lib", None)
    monkeypatch.setattr(ffi, "_LIB_PATH", str(tmp_path / "none.so"))
    i, x = torch.zeros(1, dtype=torch.int32), torch.zeros((1, 1, 128), dtype=torch.bfloat16)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        with pytest.raises(ImportError, match="none.so"):
            atflash.append_paged_kv_cache(x, x, i, i, (x[None], x[None]), i, i)
