"""CPU check of the workspace that the gradient of attention with a window asks for: a call grows by what its tokens do,
whatever the window, the sinks and the lengths of the sequences."""
import ctypes

import pytest

F32, BF16, F16 = 0, 1, 2


def _size(T, B=1, window=0, sinks=0, H=32, Hkv=8, D=128, dtype=BF16, S=None):
    import _sta_native as native
    g = native.WindowGradArgsC()
    a = g.fwd
    a.dtype, a.T, a.S, a.H, a.Hkv, a.D, a.B = dtype, T, T if S is None else S, H, Hkv, D, B
    a.window, a.sinks, a.sm_scale = window, sinks, 0.1
    if B > 1:
        a.starts = a.k_starts = ctypes.addressof(a)       # not read by the size
    n = native.lib().sta_window_grad_workspace_size(ctypes.byref(g))
    assert n > 0
    return n


def _rows(T, H=32, **_):
    return T * H * 8                                       # two numbers a row


# A record is 2 x 32 D floats a wave of its workgroup: tiles are shared out among about 1024 items in all, or the near ones
# among those and one more a tile that is shared, each a record.  1024 records of four waves and D 128 are 134 MB, a tile's own
# two records at most 16 D bytes a key and kv head, the sequences' last tiles among them.
def _bound(T, B, Hkv=8, D=128, **kw):
    return _rows(T, **kw) + 3 * 1024 * 2 * 128 * D * 4 + 4 * Hkv * (T + 128 * B) * D * 8


@pytest.mark.parametrize("T", [1024, 8192, 32768, 131072])
@pytest.mark.parametrize("window,sinks", [(128, 4), (128, 1024), (1024, 128), (128, 1 << 20), (1, 5000), (4096, 4096)])
def test_many_sinks(window, sinks, T):
    assert _size(T, window=window, sinks=sinks) <= _bound(T, 1), _size(T, window=window, sinks=sinks) / 1e6


@pytest.mark.parametrize("dtype,H,Hkv,D", [(F32, 32, 8, 64), (F16, 24, 1, 128), (BF16, 8, 8, 64), (BF16, 64, 64, 128)])
@pytest.mark.parametrize("sinks", [4, 700, 6000])
def test_doubled_tokens_take_at_most_twice_the_workspace(sinks, H, Hkv, D, dtype):
    sizes = [_size(T, window=300, sinks=sinks, H=H, Hkv=Hkv, D=D, dtype=dtype) for T in (8192, 16384, 32768, 65536)]
    for a, b in zip(sizes, sizes[1:]):
        # fewer tokens may just miss being shared out among as many items
        assert b <= 2 * a + 1024 * 2 * 128 * D * 4 * 2, [x / 1e6 for x in sizes]


@pytest.mark.parametrize("window,sinks", [(0, 0), (0, 4), (512, 4), (64, 64), (512, 0)])
@pytest.mark.parametrize("T,B", [(8192, 4096), (16384, 512), (8192, 100), (65536, 65535)])
@pytest.mark.parametrize("H,Hkv", [(32, 8), (32, 1), (8, 8)])
def test_sequences_that_share_nothing_reserve_nothing(T, B, window, sinks, H, Hkv):
    """Many short sequences: at most the records that as many tokens of few sequences may need."""
    size = _size(T, B=B, window=window, sinks=sinks, H=H, Hkv=Hkv)
    assert size <= _rows(T, H=H) + 4 * 1024 * 2 * 128 * 128 * 4, size / 1e6


def test_a_window_that_reaches_every_key_with_its_sinks_is_none():
    for window, sinks in ((128, 8192), (128, 8064), (8000, 192), (8192, 0)):
        assert _size(8192, window=window, sinks=sinks) == _size(8192), (window, sinks)
    assert _size(8192, window=128, sinks=8063) > _size(8192)
