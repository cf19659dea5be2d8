"""GPU: attention with a window where places that a row does not see hold infinities and NaN, and where sums of large
values pass the type's range on the way, against the definitions in 64 bits (bounds of window_ref.py)."""
import pytest
import torch

import window_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
NAN, INF = float("nan"), float("inf")


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    import _sta_native
    _sta_native.lib()


def _randn(seed, shape, dtype, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(DEV)


def _run(q, k, v, dout, window, sinks, starts=None, k_starts=None):
    import window_attention as wa
    q, k, v = (x.detach().requires_grad_() for x in (q, k, v))
    out, lse = wa.window_attention(q, k, v, window=window, sinks=sinks, starts=starts, k_starts=k_starts, want_lse=True)
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), dout)
    return {"out": out.detach(), "lse": lse, "dq": dq, "dk": dk, "dv": dv}


def _check(name, got, want, bound):
    err = (got.double() - want).abs()
    same = got.double() == want                # infinities
    bad = ~(err <= bound) & ~same
    assert not bad.any(), (f"{name} off by {err[bad].max().item():.3e}, bound {bound[bad].max().item():.3e}, at "
                           f"{bad.nonzero()[0].tolist()}, {int(bad.sum())} of {bad.numel()}")


# heads: 4 keep workgroups of one wave, 64 take those of four
@pytest.mark.parametrize("dtype,D", [(BF16, 128), (BF16, 64), (F16, 128), (F32, 64), (F32, 128)])
@pytest.mark.parametrize("H,Hkv", [(4, 2), (64, 64)])
@pytest.mark.parametrize("bad", [NAN, INF, -INF])
def test_keys_that_no_row_sees(bad, H, Hkv, dtype, D):
    """A prompt behind cached keys of which the window leaves the last: what lies in front of it and behind the sinks."""
    print(f"[case] window unseen keys {bad} {H} {Hkv} {dtype} {D}", flush=True)
    T, S, window, sinks = 600, 900, 77, 3
    q, k, v, dout = _randn(1, (T, H, D), dtype, 2.0), _randn(2, (S, Hkv, D), dtype), _randn(3, (S, Hkv, D), dtype), \
        _randn(4, (T, H, D), dtype)
    lost = slice(sinks, S - T - window + 1)
    k[lost], v[lost] = 0, 0
    want = ref.attention(q, k, v, window, sinks, None, None, D ** -0.5, dout)
    k[lost], v[lost] = bad, bad
    got = _run(q, k, v, dout, window, sinks)
    for name, (value, bound) in want.items():
        _check(name, got[name], value, bound)
    assert torch.all(got["dk"][lost] == 0) and torch.all(got["dv"][lost] == 0)


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (F16, 64), (F32, 128)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (50, 0), (50, 140)])
@pytest.mark.parametrize("where", ["k", "v"])
def test_a_bad_key_reaches_the_rows_that_see_it_alone(where, window, sinks, dtype, D):
    print(f"[case] window bad key {where} {window} {sinks} {dtype} {D}", flush=True)
    T, H, at = 300, 2, 131
    q, k, v, dout = (_randn(i, (T, H, D), dtype) for i in range(4))
    want = ref.attention(q, k, v, window, sinks, None, None, D ** -0.5, dout)
    (k if where == "k" else v)[at] = NAN
    got = _run(q, k, v, dout, window, sinks)
    sees = ref.visible(T, T, window, sinks, DEV)[:, at]
    for name in ("out", "dq") + (("lse",) if where == "k" else ()):
        value, bound = want[name]
        _check(name, got[name][~sees], value[~sees], bound[~sees])
        assert torch.isnan(got[name][sees]).flatten(1).any(dim=1).all(), name
    if where == "v":
        _check("lse", got["lse"], *want["lse"])


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("window,sinks", [(None, 0), (40, 2)])
def test_rows_that_see_nothing_reach_nothing(window, sinks, dtype):
    """More rows than keys: the first see none, and hold NaN in q and in the gradient."""
    print(f"[case] window blind rows {window} {sinks} {dtype}", flush=True)
    T, S, H, D = 210, 97, 2, 64
    q, k, v, dout = _randn(1, (T, H, D), dtype), _randn(2, (S, H, D), dtype), _randn(3, (S, H, D), dtype), _randn(4, (T, H, D), dtype)
    q[:T - S], dout[:T - S] = 0, 0
    want = ref.attention(q, k, v, window, sinks, None, None, D ** -0.5, dout)
    q[:T - S], dout[:T - S] = NAN, NAN
    got = _run(q, k, v, dout, window, sinks)
    for name, (value, bound) in want.items():
        _check(name, got[name], value, bound)
    assert torch.all(got["out"][:T - S] == 0) and torch.all(got["dq"][:T - S] == 0)


@pytest.mark.parametrize("dtype,most", [(BF16, 3e38), (F32, 3e38), (F16, 6e4)])
@pytest.mark.parametrize("H", [2, 64])
def test_sums_of_large_values(H, dtype, most):
    """A row's mean of 700 values near the type's largest is in range, their sum is not."""
    print(f"[case] window large values {H} {dtype}", flush=True)
    T, D = 700, 64
    q, k = _randn(1, (T, H, D), dtype), _randn(2, (T, H, D), dtype)
    v = (_randn(3, (T, H, D), F32).clamp(-1, 1) * 0.1 + 0.9).mul(most).to(dtype)
    import window_attention as wa
    out, lse = wa.window_attention(q, k, v, window=650, sinks=2, want_lse=True)
    want = ref.attention(q, k, v, 650, 2, None, None, D ** -0.5)
    _check("out", out, *want["out"])
    _check("lse", lse, *want["lse"])


def test_garbage_outside_the_sequences_keeps_the_scale_of_fp16():
    """fp16's common scale of the scores' gradients is that of the sequences: large values and infinities outside of them
    leave the gradients' bits."""
    T, H, D = 300, 2, 64
    starts = torch.tensor([20, 120, 250], dtype=torch.int32, device=DEV)
    q, k, v, dout = (_randn(i, (T, H, D), F16, 1e-3 if i == 3 else 1.0) for i in range(4))
    want = _run(q, k, v, dout, 30, 2, starts)
    for x in (v, dout):
        x[:20] = 60000.0
        x[250:] = INF
    got = _run(q, k, v, dout, 30, 2, starts)
    for name in want:
        assert torch.equal(got[name], want[name]), name
