"""CPU checks of the paged cache's entry points: what they refuse, before anything reaches a GPU."""
import ctypes

import pytest
import torch


def _host(native):
    """16-byte aligned host memory standing for device buffers: every call here is refused first."""
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 255) // 256 * 256
    return buf, p


def _cache(native, p):
    c = native.CacheC()
    c.k = c.v = c.table = c.lens = c.weight = c.pos = p
    c.dtype, c.pages, c.page_size, c.Hkv, c.D = 1, 64, 16, 8, 128
    c.k_page_stride = c.v_page_stride = 8 * 16 * 128
    c.k_head_stride = c.v_head_stride = 16 * 128
    c.k_slot_stride = c.v_slot_stride = 128
    c.weight_page_stride = c.pos_page_stride = 8 * 16
    c.weight_head_stride = c.pos_head_stride = 16
    c.table_stride, c.table_width, c.B = 512, 512, 4
    return c


def _set(a, field, value):
    obj, name = (a.cache, field[6:]) if field.startswith("cache.") else (a, field)
    setattr(obj, name, value)


CACHE_FAULTS = [("cache.D", 96, -2), ("cache.dtype", 3, -1), ("cache.page_size", 24, -2), ("cache.page_size", 0, -2),
                ("cache.page_size", 1 << 17, -2), ("cache.pages", 0, -1), ("cache.Hkv", 0, -1), ("cache.B", 0, -1),
                ("cache.B", 70000, -1), ("cache.table_width", 0, -1), ("cache.table_stride", -1, -1)]
POINTER_FAULTS = [("cache.k", None, -1), ("cache.v", None, -1), ("cache.table", None, -1), ("cache.lens", None, -1),
                  ("cache.k_slot_stride", 4, -2), ("cache.v_head_stride", -128, -2),
                  ("cache.k_page_stride", 1 << 50, -2), ("cache.weight_page_stride", -1, -2)]


def _paged(native, p):
    a = native.PagedArgsC()
    a.cache = _cache(native, p)
    a.q = a.out = p
    a.q_batch_stride, a.q_head_stride, a.q_tok_stride = 32 * 128, 128, 128
    a.H, a.Q, a.sm_scale, a.max_len = 32, 1, 0.1, 8192
    return a


@pytest.mark.parametrize("field,value,code", CACHE_FAULTS + [
    ("H", 12, -1), ("H", 0, -1), ("Q", 0, -1), ("Q", 1 << 20, -1), ("max_len", 0, -1), ("max_len", 1 << 28, -1),
    ("sm_scale", float("nan"), -1), ("sm_scale", float("inf"), -1)])
def test_attention_refuses_shapes(field, value, code):
    import _sta_native as native
    buf, p = _host(native)
    a = _paged(native, p)
    assert native.lib().sta_paged_workspace_size(ctypes.byref(a)) > 0
    _set(a, field, value)
    assert native.lib().sta_paged_workspace_size(ctypes.byref(a)) == 0
    assert native.lib().sta_paged_attention(ctypes.byref(a), None) == code
    assert len(native.lib().sta_last_error()) > 0


@pytest.mark.parametrize("field,value,code", POINTER_FAULTS + [
    ("q", None, -1), ("out", None, -1), ("q_head_stride", 3, -2), ("workspace", None, -4)])
def test_attention_refuses_pointers(field, value, code):
    import _sta_native as native
    buf, p = _host(native)
    a = _paged(native, p)
    a.workspace, a.workspace_bytes = p, 1 << 40
    _set(a, field, value)
    assert native.lib().sta_paged_attention(ctypes.byref(a), None) == code


def test_attention_refuses_a_small_workspace_and_missing_weights():
    import _sta_native as native
    buf, p = _host(native)
    a = _paged(native, p)
    n = native.lib().sta_paged_workspace_size(ctypes.byref(a))
    a.workspace, a.workspace_bytes = p, n - 1
    assert native.lib().sta_paged_attention(ctypes.byref(a), None) == -4
    a.workspace, a.workspace_bytes = p + 16, 1 << 40
    assert native.lib().sta_paged_attention(ctypes.byref(a), None) == -4
    a.workspace, a.accumulate, a.cache.weight = p, 1, None
    assert native.lib().sta_paged_attention(ctypes.byref(a), None) == -1
    assert native.lib().sta_paged_attention(None, None) == -1
    assert native.lib().sta_paged_workspace_size(None) == 0


def test_attention_workspace_sizes():
    """Short calls need none; long ones two records a run; stored scores only below 65 rows a kv head."""
    import _sta_native as native
    buf, p = _host(native)

    def size(**kw):
        a = _paged(native, p)
        for k, v in kw.items():
            setattr(a, k, v)
        return native.lib().sta_paged_workspace_size(ctypes.byref(a))
    assert size(max_len=1024) == 1
    records = 2 * 512 * 16 * (128 * 4 + 8)
    assert records <= size() < records + 1024
    scores = 4 * 32 * 8192 * 4
    assert records + scores <= size(accumulate=1) < records + scores + 4 * 32 * 4 + 1024
    assert size(accumulate=1, max_len=1024) == 4 * 32 * 1024 * 4
    # 32 queries: 128 rows in one tile, and a record a kv head
    rows = (2 * 512 + 8 * 4) * 128 * (128 * 4 + 8)
    assert rows <= size(Q=32) <= size(Q=32, accumulate=1) < rows + 4 * 32 * 32 * 4 + 2048


def _evict(native, p):
    a = native.EvictArgsC()
    a.cache = _cache(native, p)
    a.budget, a.n_global, a.n_local, a.max_len = 100, 4, 32, 8192
    a.new_lens = p + 1024
    a.workspace, a.workspace_bytes = p, 1 << 40
    return a


@pytest.mark.parametrize("field,value,code", CACHE_FAULTS + POINTER_FAULTS + [
    ("budget", 0, -1), ("n_global", -1, -1), ("n_local", -1, -1), ("max_len", 0, -1), ("cache.weight", None, -1),
    ("cache.pos", None, -1), ("new_lens", None, -1), ("workspace", None, -4), ("workspace_bytes", 8, -4)])
def test_eviction_refuses(field, value, code):
    import _sta_native as native
    buf, p = _host(native)
    a = _evict(native, p)
    _set(a, field, value)
    assert native.lib().sta_cache_evict(ctypes.byref(a), None) == code


def test_eviction_refuses_lengths_in_place_and_a_short_destination():
    import _sta_native as native
    buf, p = _host(native)
    a = _evict(native, p)
    a.new_lens = a.cache.lens
    assert native.lib().sta_cache_evict(ctypes.byref(a), None) == -1
    a = _evict(native, p)
    a.dst_table, a.dst_width, a.dst_stride = p, 6, 6          # 96 slots for 100 keys
    assert native.lib().sta_cache_evict(ctypes.byref(a), None) == -1
    assert b"dst_table" in native.lib().sta_last_error()
    assert native.lib().sta_evict_workspace_size(None) == 0


@pytest.mark.parametrize("field,value,code", CACHE_FAULTS + POINTER_FAULTS + [
    ("T", -1, -1), ("T", 5, -1), ("T", 1 << 26, -2), ("k", None, -1), ("v_tok_stride", 2, -2), ("new_lens", None, -1)])
def test_append_refuses(field, value, code):
    import _sta_native as native
    buf, p = _host(native)
    a = native.AppendArgsC()
    a.cache = _cache(native, p)
    a.k = a.v = p
    a.k_tok_stride = a.v_tok_stride = 8 * 128
    a.k_head_stride = a.v_head_stride = 128
    a.T, a.new_lens = 4, p + 1024
    _set(a, field, value)
    assert native.lib().sta_cache_append(ctypes.byref(a), None) == code


@pytest.mark.parametrize("field,value,code", [
    ("dtype", 9, -1), ("T", -1, -1), ("H", -1, -1), ("D", 100, -2), ("D", 1024, -2), ("axes", 0, -1), ("axes", 5, -1),
    ("section", (60, 0, 0, 0), -2), ("section", (72, 0, 0, 0), -2), ("section", (-8, 0, 0, 0), -1),
    ("section", (0, 0, 0, 0), -2), ("pos_type", 3, -1), ("positions", None, -1), ("inv_freq", None, -1),
    ("q", None, -1), ("k_out", None, -1), ("q_tok_stride", 3, -2)])
def test_rotary_refuses(field, value, code):
    import _sta_native as native
    buf, p = _host(native)
    a = native.RotaryArgsC()
    a.q = a.k = a.q_out = a.k_out = a.positions = a.inv_freq = p
    for x in ("q", "k", "q_out", "k_out"):
        setattr(a, x + "_tok_stride", 1024)
        setattr(a, x + "_head_stride", 128)
    a.dtype, a.T, a.H, a.Hkv, a.D, a.axes, a.rope_scale, a.pos_scale = 1, 4, 8, 8, 128, 1, 1.0, 1.0
    a.section[0] = 64
    if field == "section":
        a.section[:] = value
    else:
        setattr(a, field, value)
    assert native.lib().sta_rotary(ctypes.byref(a), None) == code
    assert native.lib().sta_rotary(None, None) == -1


def test_rotary_of_no_tokens_is_no_launch():
    import _sta_native as native
    a = native.RotaryArgsC()
    a.dtype, a.T, a.H, a.Hkv, a.D, a.axes = 1, 0, 8, 8, 128, 1
    a.section[0] = 64
    assert native.lib().sta_rotary(ctypes.byref(a), None) == 0


def test_cpu_tensors_and_wrong_types_are_refused():
    import paged_cache as pc
    x = torch.zeros(4, 8, 64)
    with pytest.raises(RuntimeError, match="HIP device"):
        pc.rotary(x, x, torch.zeros(4, dtype=torch.int32), torch.ones(32))
    with pytest.raises(RuntimeError, match="HIP device"):
        pc.PagedCache(torch.zeros(4, 2, 16, 64), torch.zeros(4, 2, 16, 64))
