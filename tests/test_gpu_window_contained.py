"""GPU: what a key that holds infinities or NaN reaches in the gradients of attention with a window: dk and dv of the keys
that a row which sees it sees too, and no others (values and bounds of window_ref.py)."""
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


def _grads(q, k, v, dout, **how):
    import window_attention as wa
    q, k, v = (x.detach().requires_grad_() for x in (q, k, v))
    return torch.autograd.grad(wa.window_attention(q, k, v, **how), (q, k, v), dout)


# heads: 2 keep workgroups of one wave, 72 and 36 take those of four
@pytest.mark.parametrize("dtype,D", [(BF16, 128), (BF16, 64), (F16, 128), (F16, 64), (F32, 128), (F32, 64)])
@pytest.mark.parametrize("H,Hkv", [(2, 1), (72, 36)])
@pytest.mark.parametrize("window,sinks,at", [(50, 0, 431), (50, 3, 431), (1, 0, 100), (20, 130, 401), (200, 2, 640)])
@pytest.mark.parametrize("where,bad", [("k", NAN), ("v", NAN), ("v", INF)])
def test_keys_that_no_row_shares_with_a_bad_one(where, bad, window, sinks, at, H, Hkv, dtype, D):
    print(f"[case] window bad key's gradients {where} {bad} {window} {sinks} {at} {H} {Hkv} {dtype} {D}", flush=True)
    T = 950
    q, k, v, dout = (_randn(i, (T, h, D), dtype) for i, h in enumerate((H, Hkv, Hkv, H)))
    want = ref.attention(q, k, v, window, sinks, None, None, D ** -0.5, dout)
    (k if where == "k" else v)[at] = bad
    _, dk, dv = _grads(q, k, v, dout, window=window, sinks=sinks)
    sees = ref.visible(T, T, window, sinks, DEV)
    apart = ~sees[sees[:, at]].any(dim=0)
    assert int(apart.sum()) > 300
    for name, got in (("dk", dk), ("dv", dv)):
        value, bound = want[name]
        err = (got.double() - value).abs()[apart]
        wrong = ~(err <= bound[apart])
        assert not wrong.any(), f"{name}: {int(wrong.sum())} of {wrong.numel()}, the largest {err[wrong].max().item():.3e}"


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("T", [131, 950])
def test_the_rows_behind_a_sequences_last_add_nothing(T, dtype):
    """A step of rows that ends past the sequence's: its last row sees a bad key, the places behind it are none."""
    print(f"[case] window bad key under the last row {T} {dtype}", flush=True)
    H, D = 4, 64
    q, k, v, dout = (_randn(i, (T, H, D), dtype) for i in range(4))
    want = ref.attention(q, k, v, 3, 0, None, None, D ** -0.5, dout)
    v[T - 1] = NAN
    _, dk, dv = _grads(q, k, v, dout, window=3, sinks=0)
    for name, got in (("dk", dk), ("dv", dv)):
        value, bound = want[name]
        assert torch.all((got.double() - value).abs()[:T - 3] <= bound[:T - 3]), name
