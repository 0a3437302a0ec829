"""The compiled binding on the CPU: refused for another torch or another version of the C
interface, and its arguments' kinds."""
import pytest
import torch

from test_serving_cpu import _lib


def _binding():
    ffi, _ = _lib()
    try:
        return ffi, ffi.binding()
    except ImportError as e:
        pytest.skip(f"binding not built: {e}")


@pytest.mark.parametrize("name,value", [("torch_version", "1.0.0"), ("version", 99)])
def test_another_version_is_refused(monkeypatch, name, value):
    ffi, b = _binding()
    monkeypatch.setattr(ffi, "_bind", None)
    monkeypatch.setattr(b, name, value)
    with pytest.raises(ImportError, match="build it again"):
        ffi.binding()


def test_what_is_no_tensor_is_refused():
    _binding()
    import atflash
    i, x = torch.zeros(1, dtype=torch.int32), torch.zeros((1, 1, 128), dtype=torch.bfloat16)
    w, c = torch.ones(128), torch.zeros((2, 64))
    with pytest.raises(TypeError, match="q must be a tensor"):
        atflash.qk_norm_rope([1], None, w, None, c, c)
    with pytest.raises(TypeError):
        atflash.qk_norm_rope(x, None, w, None, c, c, eps="small")
    with pytest.raises(TypeError, match="parents must be a tensor"):
        atflash.fork_requests([0], i, i, i[None], 16, free_pages=i, free_head=i, shared=i)
    with pytest.raises(TypeError):
        atflash.free_requests(i, i, i[None], 16.5, free_pages=i, free_head=i)
    with pytest.raises(TypeError, match="append_key must be a tensor"):
        atflash.append_paged_kv_cache(None, x, i, i, (x, x), i, i)
    with pytest.raises(ValueError, match="CUDA"):
        atflash.append_paged_kv_cache(x, x, i, i, (x, x), i, i)
