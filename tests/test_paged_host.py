"""The paged cache without a GPU: argument checks of the Python entry points and
null arguments of the C ones."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

import webgllm_b200 as wg  # noqa: E402
from webgllm_b200 import _lib, paged, q4  # noqa: E402
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


def cache(pages=6, batch=2, max_len=100, page=16):
    return paged.PagedCache(1, batch, 2, 64, pages, max_len, page_size=page, device="cpu")


def test_pages_are_handed_out_and_taken_back():
    c = cache()
    assert c.max_pages == 7 and c.max_len == 112
    c.reserve(0, 33)  # 3 pages
    c.reserve(0, 40)  # which hold 40 already
    c.reserve(1, 1)
    assert (c.table[0, :3] >= 0).all() and (c.table[0, 3:] < 0).all() and len(c.free) == 2
    held = c.table[c.table >= 0].tolist()
    assert len(set(held)) == 4
    with pytest.raises(wg.GpuError) as e:
        c.reserve(1, 65)  # 4 more: only 2 free
    assert e.value.code == _lib.WG_OUT_OF_MEMORY and len(c.free) == 2 and (c.table[1, 1:] < 0).all()
    c.release(0)
    assert len(c.free) == 5 and (c.table[0] < 0).all()
    c.reserve(1, 65)
    assert (c.table[1, :5] >= 0).all() and len(c.free) == 1
    c.release(1)
    c.release(1)
    assert sorted(c.free) == list(range(6))


def test_trim_keeps_the_window_and_the_sinks():
    c = cache(pages=7, batch=1)
    c.reserve(0, 112)
    # a row at 80 with a window of 20 sees 61..80 and the sinks 0..16
    assert c.trim(0, 80, 20, 17) == 1  # page 2 (32..47); page 3 (48..63) is still seen
    assert c.host[0][2] < 0 and all(c.host[0][i] >= 0 for i in (0, 1, 3, 4, 5, 6))
    assert c.trim(0, 80, 20, 17) == 0
    assert c.trim(0, 111, 16, 0) == 5  # pages 0, 1, 3, 4, 5; the window begins at page 6
    assert c.trim(0, 111, 0) == 0  # no window: everything is seen
    c.reserve(0, 112, start=96)
    assert len(c.free) == 6


def test_trim_past_the_table_and_with_bad_sinks():
    """A position past the table frees what it passes, and a refusal frees
    nothing: a page is never free and in the table at once."""
    c = cache(pages=9, batch=2)
    c.reserve(0, 112)
    assert c.trim(0, 1000, 16, 20) == 5  # all but the sinks' two pages
    assert (c.table[0] >= 0).tolist() == [True, True] + [False] * 5
    c.reserve(1, 112)
    held = c.table[c.table >= 0].tolist()
    assert len(set(held)) == len(held) == 9 and not c.free
    for sinks in (-1, -20, -112):
        with pytest.raises(wg.GpuError):
            c.trim(1, 60, 16, sinks)
    assert not c.free and (c.table[1] >= 0).all()


def test_cache_refusals():
    for kw in (dict(page=24), dict(page=0), dict(pages=0), dict(batch=0), dict(max_len=0)):
        with pytest.raises(wg.ShapeError):
            cache(**kw)
    with pytest.raises(wg.GpuError):
        paged.PagedCache(1, 1, 1, 64, 4, 64, dtype=torch.float32, device="cpu")
    with pytest.raises(wg.RangeError):
        cache().reserve(0, 113)


def test_native_calls_leave_what_they_do_not_take():
    """webgllm_b200._host takes CUDA tensors only; for anything else it returns
    None and Python's code says what is wrong."""
    host = q4.host_calls()
    if host is None:
        pytest.skip("webgllm_b200._host is not built")
    t = torch.zeros(2, 4, 16, 64, dtype=torch.float16)
    i = torch.zeros(2, dtype=torch.int32)
    table = torch.zeros((2, 3), dtype=torch.int32)
    assert host.attention_paged(t[:, 0], i, t, t, table, 0, 0, None, None, None) is None
    assert host.rope_kv_paged(t, i, t, t, table, 4, 1e4, None, None, 1e-5, None, None) is None
    assert host.spec_sample(torch.zeros(1, 2, 8), None, None, torch.zeros(2, 1), 1.0, None) is None
    for fn in (host.attention_paged, host.rope_kv_paged, host.spec_sample):
        assert fn() is None and fn(*[None] * 10) is None and fn(*["x"] * 12) is None and fn(*[object()] * 6) is None
