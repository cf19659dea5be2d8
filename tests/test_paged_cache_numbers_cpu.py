"""CPU checks of sizes and numbers beyond 32 bits at the paged cache's entry points, whose C structs hold 32: nothing is
launched, and tensors that would not fit here stand on the meta device."""
import ctypes

import pytest
import torch

BIG = 2 ** 32


@pytest.fixture
def native(monkeypatch):
    import _sta_native as native

    def launch(fn, args, dev, what):
        launched.append((what, args))
    launched = native_launched
    launched.clear()
    monkeypatch.setattr(native, "_device_input", lambda x, name: None)
    monkeypatch.setattr(native, "_launch", launch)
    return native


native_launched = []


def _meta(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("T", [BIG + 1, BIG, 2 ** 31])
def test_rotary_refuses_more_tokens_than_32_bits_hold(native, T):
    pos, inv = _meta(T, dtype=torch.int32), _meta(8, dtype=torch.float32)
    for q, k in ((_meta(T, 1, 16), None), (_meta(T, 1, 16), _meta(T, 2, 16))):
        with pytest.raises(ValueError, match="tokens"):
            native.rotary(q, k, pos, inv)
    assert not native_launched


def test_rotary_keeps_the_sizes_it_takes(native):
    T = 2 ** 31 - 1
    native.rotary(_meta(T, 1, 16), None, _meta(T, dtype=torch.int32), _meta(8, dtype=torch.float32))
    (_, a), = native_launched
    assert (a.T, a.H, a.Hkv, a.D, list(a.section)) == (T, 1, 0, 16, [8, 0, 0, 0])


@pytest.mark.parametrize("q,k,half,sections", [
    ((3, BIG + 4, 16), None, 8, None), ((3, 4, 16), (3, BIG + 4, 16), 8, None), ((3, 4, BIG + 16), None, 8, None),
    ((3, 4, 16), None, 8, (BIG + 8, -BIG))])
def test_rotary_does_not_fold_large_sizes_into_small_ones(native, q, k, half, sections):
    """A number that 32 bits do not hold reaches the library as one that it refuses."""
    axes = len(sections) if sections else 1
    pos, inv = _meta(axes, 3, dtype=torch.int32), _meta(half, dtype=torch.float32)
    native.rotary(_meta(*q), None if k is None else _meta(*k), pos, inv, sections)
    (_, a), = native_launched
    a.positions = a.inv_freq = 256                            # refused before any address is used
    a.q = a.q_out = a.k = a.k_out = 256
    assert native.lib().sta_rotary(ctypes.byref(a), None) in (-1, -2)


def _cache(native, pages=4, heads=2, slots=16, d=64):
    return native.PagedCache(_meta(pages, heads, slots, d), _meta(pages, heads, slots, d))


@pytest.mark.parametrize("shape", [{"heads": BIG + 2}, {"slots": BIG + 16}, {"d": BIG + 64}])
def test_a_cache_does_not_fold_large_sizes_into_small_ones(native, shape):
    c = _cache(native, **shape)
    with pytest.raises(RuntimeError):
        native.paged_attention(_meta(3, 2 * c.kv_heads, c.head_dim), c, _meta(3, 5, dtype=torch.int32),
                               _meta(3, dtype=torch.int32), max_len=64)
    assert not native_launched


@pytest.mark.parametrize("q", [(BIG + 3, 4, 64), (3, BIG + 4, 64), (3, 4, BIG + 1, 64)])
def test_attention_refuses_more_sequences_heads_or_queries(native, q):
    with pytest.raises(RuntimeError):
        native.paged_attention(_meta(*q), _cache(native), _meta(q[0], 5, dtype=torch.int32),
                               _meta(q[0], dtype=torch.int32), max_len=64)
    assert not native_launched


def test_wide_tables_and_many_pages_stay_as_large_as_they_can(native):
    c = _cache(native, pages=BIG + 4)
    assert c._c.pages == 2 ** 31 - 1
    native.paged_attention(_meta(3, 4, 64), c, _meta(3, BIG + 5, dtype=torch.int32), _meta(3, dtype=torch.int32),
                           max_len=64)
    (_, a), = native_launched
    assert a.cache.table_width == 2 ** 31 - 1 and a.max_len == 64
    evictable = native.PagedCache(c.k, c.v, _meta(BIG + 4, 2, 16, dtype=torch.float32),
                                  _meta(BIG + 4, 2, 16, dtype=torch.int32))
    native.cache_evict(evictable, _meta(3, 5, dtype=torch.int32), _meta(3, dtype=torch.int32), 64, max_len=70,
                       dst_table=_meta(3, BIG + 1, dtype=torch.int32))
    assert native_launched[1][1].dst_width == 2 ** 31 - 1


def test_index_tensors_of_64_bits_are_clamped(native):
    """A length, page or offset beyond 32 bits stays as far beyond as it can: it does not become a small one."""
    x = torch.tensor([2 ** 32 + 5, -2 ** 32 + 3, 2 ** 31, -2 ** 31 - 1, 7, -1, 2 ** 31 - 1, -2 ** 31])
    got = native._ints(x, x.device)
    most, least = 2 ** 31 - 1, -2 ** 31
    assert got.dtype == torch.int32 and got.tolist() == [most, least, most, least, 7, -1, most, least]
    table = native._ints(x.reshape(2, 4).t(), x.device)
    assert table.stride(-1) == 1 and table.tolist() == got.reshape(2, 4).t().tolist()
    same = torch.tensor([1, 2], dtype=torch.int32)
    assert native._ints(same, same.device) is same


def _append_args(native, T):
    """Arguments that are refused for k at the latest, so that nothing is launched."""
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 255) // 256 * 256
    a = native.AppendArgsC()
    c = a.cache
    c.k = c.v = c.table = c.lens = p
    c.dtype, c.pages, c.page_size, c.Hkv, c.D = 1, 64, 16, 1, 64
    for x in ("k", "v"):
        setattr(c, x + "_page_stride", 16 * 64), setattr(c, x + "_head_stride", 16 * 64), setattr(c, x + "_slot_stride", 64)
    c.table_stride, c.table_width, c.B = 4, 4, 2
    a.T, a.starts, a.new_lens = T, p, p + 1024
    return buf, a


@pytest.mark.parametrize("T,code", [(2 ** 26 - 4, -1), (2 ** 26 - 3, -2), (2 ** 26 - 1, -2)])
def test_append_takes_as_many_tokens_as_a_grid_holds(T, code):
    """Four tokens a workgroup of 256 threads: a grid holds below 2^32 threads, so 2^24 - 1 workgroups."""
    import _sta_native as native
    buf, a = _append_args(native, T)
    assert native.lib().sta_cache_append(ctypes.byref(a), None) == code


@pytest.mark.parametrize("B,Hkv,ok", [(32768, 65535, True), (32769, 65535, False), (65535, 65535, False)])
def test_eviction_numbers_its_heads_in_32_bits(B, Hkv, ok):
    """The kernel numbers the (sequence, kv head) pairs in an int."""
    import _sta_native as native
    a = native.EvictArgsC()
    c = a.cache
    c.dtype, c.pages, c.page_size, c.Hkv, c.D = 1, 4, 1, Hkv, 64
    c.table_stride, c.table_width, c.B = 1, 1, B
    a.budget, a.max_len = 1, 1
    assert (native.lib().sta_evict_workspace_size(ctypes.byref(a)) > 0) == ok
    assert ok or native.lib().sta_cache_evict(ctypes.byref(a), None) == -1


def test_workspace_of_stored_and_reformed_weights():
    """Scores are stored for fp32 and below 64 rows a kv head; from 64 on, 16-bit weights are formed again without them."""
    import _sta_native as native

    def size(H, Q, dtype, accumulate):
        a = native.PagedArgsC()
        c = a.cache
        c.dtype, c.pages, c.page_size, c.Hkv, c.D = native.DTYPES[dtype], 64, 16, 8, 64
        c.table_stride, c.table_width, c.B = 512, 512, 4
        a.H, a.Q, a.sm_scale, a.max_len, a.accumulate = H, Q, 0.1, 8192, accumulate
        return native.lib().sta_paged_workspace_size(ctypes.byref(a))
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        for H, Q in ((56, 9), (32, 16), (512, 1), (504, 1)):  # 63, 64, 64 and 63 rows a kv head
            more = size(H, Q, dtype, 1) - size(H, Q, dtype, 0)
            stats = 4 * H * 8 if Q == 1 else 0                # a maximum and a sum a row; several queries have room for them
            scores = 4 * H * Q * 8192 * 4 if dtype == torch.float32 or H // 8 * Q < 64 else 0
            assert stats + scores <= more < stats + scores + 512
