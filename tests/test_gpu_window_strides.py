"""GPU: attention with a window and its gradients on heads-first, sliced, shared and expanded tensors of sizes that take
workgroups of four waves, bit for bit what contiguous ones give; and what transforms of functions get."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
T, H, HKV = 2900, 26, 13                                   # 23 tiles of 128 rows: 598 of q, 299 of k


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    import _sta_native
    _sta_native.lib()


def _randn(seed, shape, dtype):
    g = torch.Generator(DEV).manual_seed(seed)
    return torch.randn(shape, generator=g, device=DEV, dtype=dtype)


def _run(q, k, v, dout, **how):
    import window_attention as wa
    q, k, v = (x.detach().requires_grad_() for x in (q, k, v))
    out, lse = wa.window_attention(q, k, v, want_lse=True, **how)
    return [out.detach(), lse, *torch.autograd.grad(out, (q, k, v), dout)]


def _same(got, want):
    for name, a, b in zip(("out", "lse", "dq", "dk", "dv"), got, want):
        assert torch.equal(a, b), name


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (BF16, 64), (F16, 128), (F16, 64), (F32, 128), (F32, 64)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (300, 5)])
def test_strides(window, sinks, dtype, D):
    print(f"[case] window strides {window} {sinks} {dtype} {D}", flush=True)
    starts = torch.tensor([3, 1000, 1001, 2890], dtype=torch.int32, device=DEV)
    how = dict(window=window, sinks=sinks, starts=starts)
    fused = _randn(1, (T, H + 2 * HKV, D), dtype)          # a projection of all three
    heads_first = [_randn(2 + i, (h, T, D), dtype).transpose(0, 1) for i, h in enumerate((H, HKV, HKV, H))]
    wide = _randn(8, (T, HKV, 2 * D), dtype)               # keys and values side by side
    shared = _randn(9, (T, 1, D), dtype).expand(T, HKV, D)
    dout = _randn(10, (T, H, D), dtype)
    one = torch.ones((), dtype=dtype, device=DEV).expand(T, H, D)
    for q, k, v, g in ((fused[:, :H], fused[:, H:H + HKV], fused[:, H + HKV:], heads_first[3]), (*heads_first[:3], dout),
                       (fused[:, :H], wide[..., :D], wide[..., D:], one), (heads_first[0], shared, shared, dout),
                       (fused[:, 2:H + 2], heads_first[1], wide[..., D:], wide[:, :1, :D].expand(T, H, D))):
        _same(_run(q, k, v, g, **how), _run(*(x.contiguous() for x in (q, k, v, g)), **how))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_step_between_tokens_of_many_bytes(dtype):
    """Rows far apart: the copies' offsets of up to 7 of them pass 31 bits."""
    D, n, step = 64, 40, (1 << 29) // dtype.itemsize
    free = torch.cuda.mem_get_info()[0]
    if free < (n + 1) * step * dtype.itemsize * 2:
        pytest.skip("not enough memory")
    big = torch.empty(n * step, dtype=dtype, device=DEV)
    rows = big.as_strided((n, 2, D), (step, D, 1))
    rows.copy_(_randn(3, (n, 2, D), dtype))
    q, dout = _randn(1, (n, 2, D), dtype), _randn(2, (n, 2, D), dtype)
    _same(_run(q, rows, rows, dout, window=9, sinks=2), _run(q, rows.contiguous(), rows.contiguous(), dout, window=9, sinks=2))
    _same(_run(rows, q, q, rows, window=None), _run(rows.contiguous(), q, q, rows.contiguous(), window=None))


def test_transforms_of_functions_raise():
    import paged_cache as pc
    import window_attention as wa
    q, k, v = (_randn(i, (9, 2, 64), F32) for i in range(3))
    w, pos, inv = torch.ones(64, device=DEV), torch.arange(9, dtype=torch.int32, device=DEV), torch.rand(32, device=DEV)
    for f in (lambda x: wa.window_attention(x, k, v), lambda x: wa.window_attention(q, k, x),
              lambda x: pc.norm_rotary(x, k, w, w, pos, inv)[0]):
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda x: f(x).sum())(q)
        with pytest.raises(RuntimeError):
            torch.func.vmap(f)(q[None])
        with pytest.raises(RuntimeError):
            torch.func.jvp(f, (q,), (q,))
        with pytest.raises(RuntimeError):
            torch.func.jacrev(f)(q)
    assert torch.isfinite(wa.window_attention(q, k, v)).all()      # and leave the library usable
