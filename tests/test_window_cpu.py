"""CPU checks of the normed rotation, of attention with a window and of attention behind a shared prefix: what their entry
points refuse before anything reaches a GPU, and how they take part in automatic differentiation, with formulas in place of
the launches."""
import ctypes

import pytest
import torch
import torch.autograd.forward_ad as fwad


def _host():
    """256-byte aligned host memory standing for device buffers: every call here is refused first, or launches nothing."""
    buf = ctypes.create_string_buffer(4096)
    return buf, (ctypes.addressof(buf) + 255) // 256 * 256


def _set(a, field, value):
    *path, name = field.split(".")
    for x in path:
        a = getattr(a, x)
    if name == "section":
        a.section[:] = value
    else:
        setattr(a, name, value)


# ---------------------------------------------------------------- normed rotation
def _norm(native, p, grad):
    g = native.NormRotaryGradArgsC()
    a = g.fwd
    r = a.rot
    r.q = r.k = r.q_out = r.k_out = r.positions = r.inv_freq = p
    for x in ("q", "k", "q_out", "k_out"):
        setattr(r, x + "_tok_stride", 1024)
        setattr(r, x + "_head_stride", 128)
    r.dtype, r.T, r.H, r.Hkv, r.D, r.axes, r.rope_scale, r.pos_scale = 1, 4, 8, 8, 128, 1, 1.0, 1.0
    r.section[0] = 64
    a.q_weight = a.k_weight = p
    a.weight_dtype, a.eps = 0, 1e-6
    g.dq_out = g.dk_out = g.dq_weight = g.dk_weight = g.workspace = p
    g.dq_out_tok_stride = g.dk_out_tok_stride = 1024
    g.dq_out_head_stride = g.dk_out_head_stride = 128
    g.workspace_bytes = 1 << 40
    return g if grad else a


NORM_FAULTS = [("rot.D", 516, -2), ("rot.D", 4, -2), ("rot.dtype", 3, -1), ("rot.T", -1, -1), ("rot.H", 1 << 20, -1),
               ("rot.axes", 5, -1), ("rot.section", [60, 0, 0, 0], -2), ("rot.section", [-8, 72, 0, 0], -1), ("rot.q", None, -1),
               ("rot.k_out", None, -1), ("rot.positions", None, -1), ("rot.inv_freq", None, -1), ("rot.pos_type", 7, -1),
               ("rot.q_head_stride", 4, -2), ("rot.k_tok_stride", -8, -2), ("rot.inverse", 1, -1), ("weight_dtype", 9, -1),
               ("eps", -1e-6, -1), ("eps", float("nan"), -1), ("eps", float("inf"), -1)]


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("field,value,code", NORM_FAULTS)
def test_normed_rotation_refuses(field, value, code, grad):
    import _sta_native as native
    buf, p = _host()
    a = _norm(native, p, grad)
    _set(a, "fwd." + field if grad else field, value)
    call = native.lib().sta_norm_rotary_grad if grad else native.lib().sta_norm_rotary
    assert call(ctypes.byref(a), None) == code
    assert call(None, None) == -1


@pytest.mark.parametrize("grad", [False, True])
def test_normed_rotation_refuses_weights_off_16_bytes(grad):
    import _sta_native as native
    buf, p = _host()
    a = _norm(native, p, grad)
    (a.fwd if grad else a).k_weight = p + 4
    call = native.lib().sta_norm_rotary_grad if grad else native.lib().sta_norm_rotary
    assert call(ctypes.byref(a), None) == -2


@pytest.mark.parametrize("field,value,code", [("dq_out", None, -1), ("dk_out", None, -1), ("dq_out_head_stride", 4, -2),
                                              ("dk_out_tok_stride", 1 << 50, -2), ("workspace", None, -4),
                                              ("workspace_bytes", 100, -4)])
def test_the_gradient_of_the_normed_rotation_refuses(field, value, code):
    import _sta_native as native
    buf, p = _host()
    g = _norm(native, p, True)
    assert native.lib().sta_norm_rotary_grad_workspace_size(ctypes.byref(g)) >= 2 * 128 * 4
    _set(g, field, value)
    assert native.lib().sta_norm_rotary_grad(ctypes.byref(g), None) == code


def test_normed_rotation_of_no_tokens_is_no_launch():
    import _sta_native as native
    a = native.NormRotaryArgsC()
    a.rot.dtype, a.rot.H, a.rot.Hkv, a.rot.D, a.rot.axes = 1, 8, 8, 128, 1
    a.rot.section[0] = 64
    assert native.lib().sta_norm_rotary(ctypes.byref(a), None) == 0
    g = native.NormRotaryGradArgsC()
    g.fwd = a
    assert native.lib().sta_norm_rotary_grad_workspace_size(ctypes.byref(g)) == 1
    assert native.lib().sta_norm_rotary_grad(ctypes.byref(g), None) == 0


# ---------------------------------------------------------------- attention with a window, packed
def _window(native, p, grad):
    g = native.WindowGradArgsC()
    a = g.fwd
    a.q = a.k = a.v = a.out = a.lse = a.rest = a.starts = a.k_starts = p
    for x, h in (("q", 32), ("k", 8), ("v", 8)):
        setattr(a, x + "_tok_stride", h * 128)
        setattr(a, x + "_head_stride", 128)
    a.dtype, a.T, a.S, a.H, a.Hkv, a.D, a.B, a.window, a.sinks, a.sm_scale = 1, 1000, 1000, 32, 8, 128, 3, 100, 4, 0.1
    g.dout = g.dq = g.dk = g.dv = g.workspace = p
    g.dout_tok_stride, g.dout_head_stride, g.workspace_bytes = 32 * 128, 128, 1 << 40
    return g if grad else a


SHAPE_FAULTS = [("D", 96, -2), ("D", 0, -2), ("dtype", 3, -1), ("T", -1, -1), ("S", -1, -1), ("T", (1 << 28) + 1, -1),
                ("S", (1 << 28) + 1, -1), ("H", 12, -1), ("H", 0, -1), ("Hkv", 0, -1), ("H", 65536, -1), ("B", 0, -1),
                ("B", 65536, -1), ("starts", None, -1), ("k_starts", None, -1), ("window", -1, -1), ("sinks", -1, -1),
                ("sm_scale", float("nan"), -1), ("sm_scale", float("inf"), -1), ("T", 1 << 28, -2)]


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("field,value,code", SHAPE_FAULTS + [
    ("q", None, -1), ("k", None, -1), ("v", None, -1), ("out", None, -1), ("lse", None, -1), ("q_head_stride", 4, -2),
    ("k_tok_stride", -1024, -2), ("v_tok_stride", 1 << 50, -2)])
def test_window_attention_refuses(field, value, code, grad):
    import _sta_native as native
    buf, p = _host()
    a = _window(native, p, grad)
    L = native.lib()
    if grad:
        assert L.sta_window_grad_workspace_size(ctypes.byref(a)) > 0
    _set(a, "fwd." + field if grad else field, value)
    assert (L.sta_window_attention_grad if grad else L.sta_window_attention)(ctypes.byref(a), None) == code
    if grad and (field, value, code) in SHAPE_FAULTS:
        assert L.sta_window_grad_workspace_size(ctypes.byref(a)) == 0
    assert L.sta_window_attention(None, None) == -1 and L.sta_window_attention_grad(None, None) == -1


def test_window_attention_refuses_places_off_16_bytes():
    import _sta_native as native
    buf, p = _host()
    L = native.lib()
    for field, code in (("q", -2), ("out", -1), ("rest", -2)):
        a = _window(native, p, False)
        setattr(a, field, p + 2)
        assert L.sta_window_attention(ctypes.byref(a), None) == code, field
    for field, code in (("dout", -2), ("dq", -1), ("dk", -1), ("dv", -1), ("workspace", -4)):
        a = _window(native, p, True)
        setattr(a, field, p + 2)
        assert L.sta_window_attention_grad(ctypes.byref(a), None) == code, field


def test_window_attention_refuses_token_strides_whose_copies_pass_32_bits():
    import _sta_native as native
    buf, p = _host()
    for x in ("q", "k", "v", "dout"):
        g = _window(native, p, True)
        _set(g, x + "_tok_stride" if x == "dout" else f"fwd.{x}_tok_stride", (1 << 28) + 8)      # bf16: above 2^29 bytes
        assert native.lib().sta_window_attention_grad(ctypes.byref(g), None) == -2, x
        if x != "dout":
            assert native.lib().sta_window_attention(ctypes.byref(g.fwd), None) == -2, x


@pytest.mark.parametrize("field,value,code", [("dout", None, -1), ("dq", None, -1), ("dk", None, -1), ("dv", None, -1),
                                              ("dout_head_stride", 4, -2), ("workspace", None, -4),
                                              ("workspace_bytes", 1000, -4)])
def test_the_gradient_of_window_attention_refuses(field, value, code):
    import _sta_native as native
    buf, p = _host()
    g = _window(native, p, True)
    _set(g, field, value)
    assert native.lib().sta_window_attention_grad(ctypes.byref(g), None) == code


def test_window_attention_without_queries_is_no_launch():
    import _sta_native as native
    a = native.WindowArgsC()
    a.dtype, a.H, a.Hkv, a.D, a.B = 1, 8, 8, 64, 1
    assert native.lib().sta_window_attention(ctypes.byref(a), None) == 0


def test_window_workspace_holds_two_numbers_a_row_and_the_records():
    import _sta_native as native
    buf, p = _host()
    g = _window(native, p, True)

    def size(**kw):
        for name, value in kw.items():
            setattr(g.fwd, name, value)
        return native.lib().sta_window_grad_workspace_size(ctypes.byref(g))
    rows = 8192 * 32 * 8
    # many tiles and no sinks: none is shared out, so that there are no records
    assert size(T=8192, S=8192, window=1024, sinks=0) == rows
    assert size(sinks=4) > rows
    # a window that reaches every key is none, and needs no record for its sinks
    assert size(window=8192, sinks=4) == size(window=0, sinks=0)


# ---------------------------------------------------------------- the paged forms
def _paged(native, p, a):
    c = a.cache
    c.k = c.v = c.table = c.lens = p
    c.dtype, c.pages, c.page_size, c.Hkv, c.D = 1, 64, 16, 8, 128
    c.k_page_stride = c.v_page_stride = 8 * 16 * 128
    c.k_head_stride = c.v_head_stride = 16 * 128
    c.k_slot_stride = c.v_slot_stride = 128
    c.table_stride, c.table_width, c.B = 512, 512, 4
    a.q = a.out = a.workspace = p
    a.q_batch_stride, a.q_head_stride, a.q_tok_stride = 32 * 128, 128, 128
    a.H, a.Q, a.sm_scale, a.max_len, a.workspace_bytes = 32, 1, 0.1, 8192, 1 << 40


PAGED_FAULTS = [("cache.D", 96, -2), ("cache.page_size", 24, -2), ("cache.B", 0, -1), ("H", 12, -1), ("Q", 0, -1),
                ("max_len", 0, -1), ("sm_scale", float("nan"), -1), ("accumulate", 1, -2)]
PAGED_PLACES = [("q", None, -1), ("out", None, -1), ("cache.k", None, -1), ("cache.table", None, -1),
                ("q_head_stride", 4, -2), ("workspace", None, -4), ("workspace_bytes", 100, -4)]


@pytest.mark.parametrize("form", ["paged", "own"])
@pytest.mark.parametrize("field,value,code", PAGED_FAULTS + PAGED_PLACES)
def test_paged_forms_refuse_as_paged_attention(field, value, code, form):
    import _sta_native as native
    buf, p = _host()
    L = native.lib()
    if form == "paged":
        a, size, call = native.PagedWindowArgsC(), L.sta_paged_window_workspace_size, L.sta_paged_window_attention
        a.window, a.sinks = 2000, 4
    else:
        a, size, call = native.PrefixArgsC(), L.sta_prefix_workspace_size, L.sta_prefix_attention
        a.prefix, a.prefix_width, a.prefix_len = p, 32, 500
    _paged(native, p, getattr(a, form))
    assert size(ctypes.byref(a)) > 1
    _set(a, f"{form}.{field}", value)
    assert call(ctypes.byref(a), None) == code
    if (field, value, code) in PAGED_FAULTS:
        assert size(ctypes.byref(a)) == 0
    assert call(None, None) == -1


@pytest.mark.parametrize("field,value,code", [("window", -1, -1), ("sinks", -1, -1)])
def test_paged_window_refuses(field, value, code):
    import _sta_native as native
    buf, p = _host()
    a = native.PagedWindowArgsC()
    _paged(native, p, a.paged)
    a.window, a.sinks = 2000, 4
    setattr(a, field, value)
    assert native.lib().sta_paged_window_attention(ctypes.byref(a), None) == code


def test_a_paged_window_needs_the_workspace_of_the_keys_that_it_sees():
    import _sta_native as native
    buf, p = _host()
    a = native.PagedWindowArgsC()
    _paged(native, p, a.paged)
    L = native.lib()
    sizes = []
    for a.window in (100, 2000, 1 << 27):
        sizes.append(L.sta_paged_window_workspace_size(ctypes.byref(a)))
    assert 0 < sizes[0] <= sizes[1] <= sizes[2] == L.sta_paged_workspace_size(ctypes.byref(a.paged))


@pytest.mark.parametrize("field,value,code", [("prefix", None, -1), ("prefix_width", 0, -1), ("prefix_len", 0, -1),
                                              ("prefix_len", 513, -1), ("prefix_len", 1 << 28, -1), ("own.cache.B", 60000, -1)])
def test_prefix_refuses(field, value, code):
    import _sta_native as native
    buf, p = _host()
    a = native.PrefixArgsC()
    _paged(native, p, a.own)
    a.prefix, a.prefix_width, a.prefix_len, a.own.Q, a.own.q_tok_stride = p, 32, 512, 4, 128
    a.own.q_head_stride, a.own.q_batch_stride = 4 * 128, 32 * 4 * 128
    _set(a, field, value)
    assert native.lib().sta_prefix_attention(ctypes.byref(a), None) == code


# ---------------------------------------------------------------- Python
def test_cpu_tensors_are_refused():
    import paged_cache as pc
    import window_attention as wa
    x = torch.zeros(4, 8, 64)
    with pytest.raises(RuntimeError, match="HIP device"):
        wa.window_attention(x, x, x)
    with pytest.raises(RuntimeError, match="HIP device"):
        wa.window_attention_grad(x, x, x, x, x, torch.zeros(4, 8))
    with pytest.raises(RuntimeError, match="HIP device"):
        pc.norm_rotary(x, x, None, None, torch.zeros(4, dtype=torch.int32), torch.ones(32))
    with pytest.raises(RuntimeError, match="HIP device"):
        pc.norm_rotary_grad(x, x, x, x, None, None, torch.zeros(4, dtype=torch.int32), torch.ones(32))


@pytest.fixture
def filled(monkeypatch):
    """The calls with CPU tensors up to the launch, which gets the arguments."""
    import _sta_native as native
    calls = []
    monkeypatch.setattr(native, "_device_input", lambda x, name: None)
    monkeypatch.setattr(native, "_launch", lambda fn, args, dev, what: calls.append((what, args)))
    return native, calls


def test_window_arguments(filled):
    import window_attention as wa
    native, calls = filled
    q, k = torch.zeros(10, 4, 64), torch.zeros(10, 2, 64)
    starts = torch.tensor([0, 3, 10], dtype=torch.int32)
    for bad, kw in ((ValueError, dict(window=0)), (ValueError, dict(window=-5)), (ValueError, dict(k_starts=starts)),
                    (ValueError, dict(starts=starts[:1])), (ValueError, dict(starts=starts[None])),
                    (ValueError, dict(starts=starts, k_starts=starts[:2]))):
        with pytest.raises(bad):
            wa.window_attention(q, k, k, **kw)
    for args in ((q, k, k[:9]), (q, k, k[..., :32]), (q[0], k, k), (q[..., :32], k, k)):
        with pytest.raises(ValueError):
            wa.window_attention(*args)
    with pytest.raises(ValueError, match="k_starts"):
        wa.window_attention(q, k[:9], k[:9], starts=starts)
    with pytest.raises(TypeError):
        wa.window_attention(q, k.half(), k)
    assert not calls
    fused = torch.zeros(10, 8, 64)
    wa.window_attention(fused[:, :4], fused[:, 4:6], fused[:, 6:], window=1 << 40, sinks=2, starts=starts)
    what, a = calls.pop()
    assert what == "sta_window_attention" and (a.T, a.S, a.H, a.Hkv, a.D, a.B) == (10, 10, 4, 2, 64, 2)
    assert (a.q_tok_stride, a.k_tok_stride, a.k_head_stride) == (512, 512, 64) and a.k == fused.data_ptr() + 4 * 64 * 4
    assert a.window == 2 ** 31 - 1 and a.sinks == 2 and a.rest is None and abs(a.sm_scale - 0.125) < 1e-9


def test_window_gradient_arguments(filled):
    import window_attention as wa
    q, k, lse = torch.zeros(10, 4, 64).bfloat16(), torch.zeros(10, 2, 64).bfloat16(), torch.zeros(10, 4)
    for bad, args in ((ValueError, (q[:9], q, k, k, q, lse)), (TypeError, (q.float(), q, k, k, q, lse)),
                      (ValueError, (q, q, k, k, q[:, :2], lse)), (ValueError, (q, q, k, k, q, lse.t())),
                      (ValueError, (q, q, k, k, q, lse.double())), (TypeError, (q, q, k, k, q, lse, q.float()))):
        with pytest.raises(bad):
            wa.window_attention_grad(*args)


def test_normed_rotation_arguments(filled):
    import paged_cache as pc
    native, calls = filled
    q, k, w = torch.zeros(5, 4, 64), torch.zeros(5, 2, 64), torch.ones(64)
    pos, inv = torch.arange(5, dtype=torch.int32), torch.ones(32)
    for bad, args in ((ValueError, (q, k, w[:32], w, pos, inv)), (TypeError, (q, k, w, w.half(), pos, inv)),
                      (TypeError, (q, k, w.int(), None, pos, inv)), (ValueError, (q, None, w, w, pos, inv)),
                      (ValueError, (q, k[:4], w, w, pos, inv)), (TypeError, (q, k.half(), w, w, pos, inv)),
                      (ValueError, (q, k, w, w, pos[:4], inv))):
        with pytest.raises(bad):
            pc.norm_rotary(*args)
    for bad, args in ((ValueError, (q, None, q, k, w, w, pos, inv)), (ValueError, (q[:4], k, q, k, w, w, pos, inv)),
                      (TypeError, (q.half(), k, q, k, w, w, pos, inv))):
        with pytest.raises(bad):
            pc.norm_rotary_grad(*args)
    assert not calls


# formulas in place of the launches, in float64
def _attend(q, k, v, window, sinks, starts, sm_scale):
    T = q.shape[0]
    p, j = torch.arange(T)[:, None], torch.arange(T)[None]
    seq = torch.bucketize(torch.arange(T), starts[1:].long(), right=True)
    sees = (j <= p) & ((j > p - window) | (j - starts[seq][None] < sinks)) & (seq[:, None] == seq[None])
    g = q.shape[1] // k.shape[1]
    s = torch.einsum("thd,shd->hts", q, k.repeat_interleave(g, 1)) * sm_scale
    s = s.masked_fill(~sees, float("-inf"))
    return torch.einsum("hts,shd->thd", s.softmax(-1), v.repeat_interleave(g, 1)), s.logsumexp(-1)


@pytest.fixture
def formulas(monkeypatch):
    import _sta_native as native

    def window_attention(q, k, v, window, sinks, starts, k_starts, sm_scale, want_rest=False):
        assert all(type(x) is torch.Tensor and not x.requires_grad for x in (q, k, v)) or not torch.is_grad_enabled()
        out, lse = _attend(q, k, v, window, sinks, starts, sm_scale)
        return out, lse, torch.zeros_like(out) if want_rest else None

    def window_attention_grad(dout, q, k, v, out, lse, rest, window, sinks, starts, k_starts, sm_scale):
        assert lse.shape == (q.shape[1], q.shape[0])
        with torch.enable_grad():
            x = [t.detach().requires_grad_() for t in (q, k, v)]
            return torch.autograd.grad(_attend(*x, window, sinks, starts, sm_scale)[0], x, dout)

    def formula(q, k, qw, kw, positions, inv_freq, eps):
        def turn(x, w):
            if x is None:
                return None
            n = inv_freq.numel()
            x = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps) * (1.0 if w is None else w)
            c, s = (f(positions[:, None] * inv_freq)[:, None] for f in (torch.cos, torch.sin))
            a, b = x[..., :n], x[..., n:2 * n]
            return torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * n:]], -1)
        return turn(q, qw), turn(k, kw)

    def norm_rotary(q, k, qw, kw, positions, inv_freq, sections, eps, pos_scale, rope_scale):
        return formula(q, k, qw, kw, positions, inv_freq, eps)

    def norm_rotary_grad(dq, dk, q, k, qw, kw, positions, inv_freq, sections, eps, pos_scale, rope_scale, want=True):
        x = [None if t is None else t.detach().requires_grad_() for t in (q, k, qw, kw)]
        with torch.enable_grad():
            out = formula(*x, positions, inv_freq, eps)
            pairs = [(o, d) for o, d in zip(out, (dq, dk)) if o is not None]
            got = iter(torch.autograd.grad([o for o, _ in pairs], [t for t in x if t is not None], [d for _, d in pairs]))
        got = [None if t is None else next(got) for t in x]
        return (*got[:2], *(got[2:] if want else (None, None)))
    for f in (window_attention, window_attention_grad, norm_rotary, norm_rotary_grad):
        monkeypatch.setattr(native, f.__name__, f)


def _packed(D=8):
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn((9, h, D), generator=g, dtype=torch.float64, requires_grad=True) for h in (4, 2, 2))
    return q, k, v, torch.tensor([0, 4, 9], dtype=torch.int32)


def test_window_attention_in_autograd(formulas):
    import window_attention as wa
    q, k, v, starts = _packed()
    call = lambda *x: wa.window_attention(*x, window=3, sinks=1, starts=starts, sm_scale=0.3)     # noqa: E731
    assert torch.autograd.gradcheck(call, (q, k, v))
    out, lse, rest = wa.window_attention(q, k, v, window=3, sinks=1, starts=starts, sm_scale=0.3, want_lse=True, want_rest=True)
    assert out.requires_grad and not lse.requires_grad and not rest.requires_grad and lse.shape == (9, 4)
    g = torch.ones_like(out)
    want = torch.autograd.grad(out, (q, k, v), g)
    got = wa.window_attention_grad(g, q, k, v, out, lse, rest, window=3, sinks=1, starts=starts, sm_scale=0.3)
    for a, b in zip(got, want):
        assert torch.equal(a, b) and not a.requires_grad
    once = torch.autograd.grad(call(q, k, v).square().sum(), q, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="once"):
        once.sum().backward()
    with torch.no_grad():
        assert not call(q, k, v).requires_grad


def test_normed_rotation_in_autograd(formulas):
    import paged_cache as pc
    q, k, _, _ = _packed()
    qw, kw = (torch.rand(8, dtype=torch.float64, requires_grad=True) for _ in range(2))
    pos, inv = torch.arange(9.0, dtype=torch.float64), torch.rand(4, dtype=torch.float64)
    assert torch.autograd.gradcheck(lambda *x: pc.norm_rotary(*x, pos, inv), (q, k, qw, kw))
    assert torch.autograd.gradcheck(lambda a, w: pc.norm_rotary(a, None, w, None, pos, inv)[0], (q, qw))
    assert torch.autograd.gradcheck(lambda a, b: pc.norm_rotary(a, b, None, None, pos, inv), (q, k))
    a, b = pc.norm_rotary(q, k, qw, kw, pos, inv)
    only = torch.autograd.grad(b.sum(), (q, k, qw, kw), retain_graph=True)      # q's output takes no part
    assert torch.all(only[0] == 0) and torch.all(only[2] == 0) and torch.any(only[3] != 0)
    once = torch.autograd.grad(a.square().sum(), q, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="once"):
        once.sum().backward()


def test_forward_mode_is_refused(formulas):
    import paged_cache as pc
    import window_attention as wa
    q, k, v, starts = (x.detach() for x in _packed())
    w, pos, inv = torch.ones(8, dtype=torch.float64), torch.arange(9.0, dtype=torch.float64), torch.rand(4, dtype=torch.float64)
    kw = dict(window=3, starts=starts, sm_scale=0.3)
    with fwad.dual_level():
        dual = lambda x: fwad.make_dual(x, torch.ones_like(x))                  # noqa: E731
        out, lse = wa.window_attention(q, k, v, want_lse=True, **kw)            # none of them has a tangent
        for args in ((dual(q), k, v), (q, dual(k), v), (q, k, dual(v))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                wa.window_attention(*args, **kw)
            with pytest.raises(RuntimeError, match="forward-mode"):
                wa.window_attention_grad(out, *args, out, lse, **kw)
        pc.norm_rotary(q, k, w, None, pos, inv)
        for args in ((dual(q), k, w, w), (q, dual(k), w, w), (q, k, dual(w), w), (q, k, w, dual(w))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                pc.norm_rotary(*args, pos, inv)
            with pytest.raises(RuntimeError, match="forward-mode"):
                pc.norm_rotary_grad(q, k, *args, pos, inv)
