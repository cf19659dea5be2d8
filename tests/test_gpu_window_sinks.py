"""GPU: attention with a window and many sinks, whose key tiles are shared out in steps of their own, against the
definitions in 64 bits (window_ref.py)."""
import pytest
import torch

import window_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    import _sta_native
    _sta_native.lib()


def _randn(seed, shape, dtype, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(DEV)


def _run(q, k, v, dout, window, sinks, starts=None):
    import window_attention as wa
    q, k, v = (x.detach().requires_grad_() for x in (q, k, v))
    out, lse = wa.window_attention(q, k, v, window=window, sinks=sinks, starts=starts, want_lse=True)
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), dout)
    return {"out": out.detach(), "lse": lse, "dq": dq, "dk": dk, "dv": dv}


def _inputs(T, H, Hkv, D, dtype):
    return [_randn(i, (T, h, D), dtype) for i, h in enumerate((H, Hkv, Hkv, H))]


# one wave a workgroup, then four: the steps of tiles with sinks are several times those of the others
@pytest.mark.parametrize("dtype,D", [(BF16, 128), (F16, 64), (F32, 64)])
@pytest.mark.parametrize("H,Hkv,lens,window,sinks", [(8, 2, [1900], 33, 1500), (8, 1, [1200, 40, 0, 900], 20, 700),
                                                     (52, 26, [1300], 20, 600), (26, 26, [1, 1500, 300], 5, 1000)])
def test_many_sinks(H, Hkv, lens, window, sinks, dtype, D):
    print(f"[case] window many sinks {H} {Hkv} {lens} {window} {sinks} {dtype} {D}", flush=True)
    starts = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=DEV)
    x = _inputs(sum(lens), H, Hkv, D, dtype)
    got = _run(*x, window, sinks, starts)
    want = ref.attention(*x[:3], window, sinks, starts.tolist(), None, D ** -0.5, x[3])
    for name, (value, bound) in want.items():
        err = (got[name].double() - value).abs()
        bad = ~(err <= bound) & ~(got[name].double() == value)
        assert not bad.any(), f"{name} off by {err[bad].max().item():.3e}, bound {bound[bad].max().item():.3e}"


def test_many_short_sequences_and_a_long_one():
    """More sequences than share a tile, one of them long: the records are the long one's."""
    g = torch.Generator().manual_seed(5)
    lens = torch.randint(0, 7, (500,), generator=g).tolist() + [1400] + torch.randint(0, 40, (60,), generator=g).tolist()
    starts = torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32, device=DEV)
    x = _inputs(sum(lens), 4, 1, 64, BF16)
    for window, sinks in ((17, 3), (None, 0), (9, 900)):
        print(f"[case] window many short sequences {window} {sinks}", flush=True)
        got = _run(*x, window, sinks, starts)
        want = ref.attention(*x[:3], window, sinks, starts.tolist(), None, 64 ** -0.5, x[3])
        for name, (value, bound) in want.items():
            err = (got[name].double() - value).abs()
            assert torch.all((err <= bound) | (got[name].double() == value)), name


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_sinks_that_reach_the_window_are_plain_causal(dtype):
    x = _inputs(700, 4, 2, 64, dtype)
    want = _run(*x, None, 0)
    for window, sinks in ((100, 600), (100, 700), (1, 1 << 30), (699, 1)):
        got = _run(*x, window, sinks)
        for name in want:
            assert torch.equal(got[name], want[name]), (name, window, sinks)
