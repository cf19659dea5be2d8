"""CPU check of the strides that attention with a window takes: token strides up to 2^29 bytes, as include/sta.h says, and head
strides of tensors with the heads first and many tokens."""
import ctypes

import pytest


def _args(native, p, dtype):
    g = native.WindowGradArgsC()
    a = g.fwd
    a.q = a.k = a.v = a.out = a.lse = a.rest = p
    for x, h in (("q", 32), ("k", 8), ("v", 8)):
        setattr(a, x + "_tok_stride", h * 128)
        setattr(a, x + "_head_stride", 128)
    a.dtype, a.T, a.S, a.H, a.Hkv, a.D, a.B, a.window, a.sinks, a.sm_scale = dtype, 1000, 1000, 32, 8, 128, 1, 100, 4, 0.1
    g.dout = g.dq = g.dk = g.dv = p
    g.dout_tok_stride, g.dout_head_stride = 32 * 128, 128
    return g                                               # no workspace: a call that is else in order returns -4


@pytest.mark.parametrize("dtype,size", [(0, 4), (1, 2), (2, 2)])
@pytest.mark.parametrize("x", ["q", "k", "v", "dout"])
def test_limits(x, dtype, size):
    import _sta_native as native
    buf = ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 255) // 256 * 256

    def call(what, value):
        g = _args(native, p, dtype)
        setattr(g if x == "dout" else g.fwd, f"{x}_{what}_stride", value)
        return native.lib().sta_window_attention_grad(ctypes.byref(g), None)
    assert call("tok", (1 << 29) // size) == -4
    assert call("tok", (1 << 29) // size + 8) == -2
    assert call("head", (1 << 28) * 128) == -4             # (heads, 2^28 tokens, 128)
    assert call("head", 1 << 44) == -2 and call("head", -8) == -2
