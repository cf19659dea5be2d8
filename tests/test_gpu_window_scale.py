"""GPU: fp16's gradients of attention with a window keep the accuracy that a sequence, a head or a far place has alone, whatever
large values the others hold (values and bounds of window_ref.py, formed of the part alone)."""
import pytest
import torch

import window_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16 = torch.float16


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    import _sta_native
    _sta_native.lib()


def _randn(seed, shape, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(F16).to(DEV)


def _grads(q, k, v, dout, **how):
    import window_attention as wa
    q, k, v = (x.detach().requires_grad_() for x in (q, k, v))
    return dict(zip(("dq", "dk", "dv"), torch.autograd.grad(wa.window_attention(q, k, v, **how), (q, k, v), dout)))


def _check(name, got, want, bound):
    err = (got.double() - want).abs()
    bad = ~(err <= bound)
    assert not bad.any(), (f"{name} off by {err[bad].max().item():.3e}, bound {bound[bad].max().item():.3e}, "
                           f"{int(bad.sum())} of {bad.numel()}")


# heads: 4 / 2 keep workgroups of one wave, 64 / 32 take those of four
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,Hkv", [(4, 2), (64, 32)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (200, 3)])
def test_sequences_beside_one_of_large_values(window, sinks, H, Hkv, D):
    print(f"[case] window fp16 beside a large sequence {window} {sinks} {H} {Hkv} {D}", flush=True)
    lens = [300, 640, 97]
    starts = torch.tensor([0, 300, 940, 1037], dtype=torch.int32, device=DEV)
    q, k, v, dout = (_randn(i, (sum(lens), h, D)) for i, h in enumerate((H, Hkv, Hkv, H)))
    v[300:940] *= 1000
    dout[300:940] *= 1000
    got = _grads(q, k, v, dout, window=window, sinks=sinks, starts=starts)
    for a, b in ((0, 300), (940, 1037)):
        want = ref.attention(q[a:b], k[a:b], v[a:b], window, sinks, None, None, D ** -0.5, dout[a:b])
        for name, x in got.items():
            _check(name, x[a:b], *want[name])


@pytest.mark.parametrize("H,Hkv", [(4, 2), (64, 32)])
def test_heads_beside_one_of_large_values(H, Hkv):
    """One row of one head, one key of another kv head."""
    print(f"[case] window fp16 beside a large head {H} {Hkv}", flush=True)
    T, D = 700, 64
    q, k, v, dout = (_randn(i, (T, h, D)) for i, h in enumerate((H, Hkv, Hkv, H)))
    dout[20, 0] *= 5000
    v[3, 1] *= 5000
    got = _grads(q, k, v, dout)
    G = H // Hkv
    for hk in range(2, Hkv) if Hkv > 2 else ():
        heads = slice(hk * G, (hk + 1) * G)
        want = ref.attention(q[:, heads], k[:, hk:hk + 1], v[:, hk:hk + 1], None, 0, None, None, D ** -0.5, dout[:, heads])
        _check("dq", got["dq"][:, heads], *want["dq"])
        for name in ("dk", "dv"):
            _check(name, got[name][:, hk:hk + 1], *want[name])
    # the two heads themselves: one has the large row, the other the large key, neither both
    for hk in (0, 1):
        heads = slice(hk * G, (hk + 1) * G)
        want = ref.attention(q[:, heads], k[:, hk:hk + 1], v[:, hk:hk + 1], None, 0, None, None, D ** -0.5, dout[:, heads])
        _check("dq", got["dq"][:, heads], *want["dq"])
        for name in ("dk", "dv"):
            _check(name, got[name][:, hk:hk + 1], *want[name])


@pytest.mark.parametrize("H", [2, 64])
def test_rows_and_keys_behind_a_window_of_large_values(H):
    """Large values in the first rows and keys: those from 50 behind 600 on do not see them, and come out as alone."""
    print(f"[case] window fp16 far from large values {H}", flush=True)
    T, D, window, at = 1500, 64, 50, 1200
    q, k, v, dout = (_randn(i, (T, H, D)) for i in range(4))
    v[:600] *= 1000
    dout[:600] *= 1000
    got = _grads(q, k, v, dout, window=window)
    # from the row `at` - window on as a sequence of its own: rows and keys from `at` on see what they see here
    a = at - window
    want = ref.attention(q[a:], k[a:], v[a:], window, 0, None, None, D ** -0.5, dout[a:])
    for name, x in got.items():
        _check(name, x[at:], want[name][0][window:], want[name][1][window:])


def test_gradients_of_all_sizes_in_one_row_range():
    """Rows of gradients from 6e-5 to 3000, each in its own sequence, in one call."""
    sizes = (6e-5, 1e-3, 1.0, 60.0, 3000.0)
    starts = torch.tensor([0, 64, 130, 190, 300, 411], dtype=torch.int32, device=DEV)
    q, k, v, dout = (_randn(i, (411, 2, 128)) for i in range(4))
    for (a, b), s in zip(ref.spans(starts.tolist(), 411), sizes):
        dout[a:b] = _randn(9, (b - a, 2, 128), s)
    got = _grads(q, k, v, dout, starts=starts)
    for a, b in ref.spans(starts.tolist(), 411):
        want = ref.attention(q[a:b], k[a:b], v[a:b], None, 0, None, None, 128 ** -0.5, dout[a:b])
        for name, x in got.items():
            _check(name, x[a:b], *want[name])
