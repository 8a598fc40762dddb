"""The paged cache without a GPU: argument checks of the Python entry points and
null arguments of the C ones."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

import webgllm_b200 as wg  # noqa: E402
from webgllm_b200 import _lib, paged  # noqa: E402
from webgllm_b200.speculative import spec_sample  # noqa: E402


def tensors(dtype=torch.float16):
    k = torch.zeros((4, 2, 16, 64), dtype=dtype)
    return (torch.zeros((2, 4, 64), dtype=dtype), torch.zeros(2, dtype=torch.int32), k, torch.zeros_like(k),
            torch.zeros((2, 2), dtype=torch.int32))


def test_c_entry_points_reject_a_null_context():
    L = _lib.lib()
    kv = _lib.wg_paged_kv()
    assert L.wg_paged_attention(None, None, 1, 1, None, 1, 1, 64, None, ctypes.byref(kv), 0, 0, None, None, 0) \
        == _lib.WG_INVALID_ARGUMENT
    assert L.wg_paged_rope_kv(None, None, 1, 1, None, 1, 1, 64, None, 1e4, None, None, 1e-5, None, ctypes.byref(kv)) \
        == _lib.WG_INVALID_ARGUMENT
    assert L.wg_paged_attention_workspace(None, 64, ctypes.byref(ctypes.c_size_t())) == _lib.WG_INVALID_ARGUMENT
    assert L.wg_spec_sample(None, None, None, None, 1, 0, 8, 1.0, None, None, None, 0) == _lib.WG_INVALID_ARGUMENT


def test_host_tensors_are_refused():
    q, pos, k, v, table = tensors()
    with pytest.raises(wg.GpuError, match="CUDA"):
        paged.attention_paged(q, pos, k, v, table)
    with pytest.raises(wg.GpuError, match="CUDA"):
        paged.rope_kv_paged(torch.zeros((2, 8 * 64)), pos, k, v, table, heads=4)
    with pytest.raises(wg.ShapeError):
        spec_sample(torch.zeros((1, 2, 8)), None, None, torch.zeros((2, 1)))


def test_cache_shapes_are_checked_before_the_device():
    q, pos, k, v, table = tensors()
    with pytest.raises(wg.ShapeError):
        paged.attention_paged(q, pos, k, v[:3], table)
    with pytest.raises(wg.ShapeError):
        paged.attention_paged(q, pos, k[0], v[0], table)
    with pytest.raises(wg.ShapeError):
        paged.attention_paged(q, pos, k, v.transpose(1, 2).contiguous().transpose(1, 2), table)
    with pytest.raises(wg.GpuError):
        paged.attention_paged(q.float(), pos, k.float(), v.float(), table)
    with pytest.raises(wg.GpuError):
        paged.attention_paged(q, pos, k, v.bfloat16(), table)
