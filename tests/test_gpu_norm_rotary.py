"""GPU: norm and rotation of queries and keys in one pass, and its gradients, against the definitions in 64 bits with
the bounds derived in norm_ref.py."""
import pytest
import torch

import norm_ref as ref

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


def _check(name, got, want):
    value, bound = want
    err = (got.double().cpu() - value).abs()
    bad = ~(err <= bound)
    assert not bad.any(), f"{name} off by {err[bad].max().item():.3e}, bound {bound[bad].max().item():.3e}, {int(bad.sum())}"


def _setup(T, H, Hkv, D, sections, dtype, weight, scale=2.0):
    half = sum(sections)
    q, k = _randn(1, (T, H, D), dtype, scale), _randn(2, (T, Hkv, D), dtype, scale)
    wq, wk = (None, None) if weight is None else (1 + _randn(3, (D,), F32, 0.3)).to(weight), (1 + _randn(4, (D,), F32, 0.3)).to(weight)
    if weight is None:
        wq = wk = None
    inv_freq = (10000.0 ** -(torch.arange(half, dtype=torch.float64) / half)).float().to(DEV)
    positions = torch.randint(0, 1 << 20, (len(sections), T), generator=torch.Generator().manual_seed(5),
                              dtype=torch.int32).to(DEV)
    return q, k, wq, wk, positions, inv_freq, sections


SHAPES = [(1, 8, 2, 128, (64,), BF16, BF16), (37, 5, 1, 128, (16, 24, 24), BF16, F32), (300, 4, 4, 64, (32,), F16, F16),
          (65, 3, 3, 80, (8, 16, 16), F32, F32), (1025, 2, 2, 64, (8, 24), F32, None), (33, 1, 7, 16, (8,), F16, None),
          (9, 40, 8, 128, (32,), BF16, BF16), (5, 2, 2, 512, (256,), F32, F32), (2100, 3, 1, 24, (8,), BF16, F16),
          (700, 1, 60, 128, (64,), F16, BF16), (4, 6, 2, 264, (8,), BF16, F32)]


@pytest.mark.parametrize("T,H,Hkv,D,sections,dtype,weight", SHAPES)
def test_forward_and_gradients(T, H, Hkv, D, sections, dtype, weight):
    import paged_cache as pc
    print(f"[case] norm rotary {T} {H} {Hkv} {D} {sections} {dtype} {weight}", flush=True)
    q, k, wq, wk, positions, inv_freq, sections = _setup(T, H, Hkv, D, sections, dtype, weight)
    how = dict(sections=sections, eps=1e-5, pos_scale=0.25, rope_scale=1.5)
    y, z = pc.norm_rotary(q, k, wq, wk, positions, inv_freq, **how)
    args = (positions, inv_freq, sections, 1e-5, 0.25, 1.5)
    _check("q", y, ref.forward(q, wq, *args))
    _check("k", z, ref.forward(k, wk, *args))
    dq, dk = _randn(6, q.shape, dtype), _randn(7, k.shape, dtype)
    got = pc.norm_rotary_grad(dq, dk, q, k, wq, wk, positions, inv_freq, **how)
    for name, d, x, w, gx, gw in (("q", dq, q, wq, got[0], got[2]), ("k", dk, k, wk, got[1], got[3])):
        want = ref.gradients(d, x, w, *args)
        _check("d" + name, gx, want[0])
        if w is None:
            assert gw is None
        else:
            assert gw.dtype == w.dtype
            _check(f"d{name}_weight", gw, want[1])
    again = pc.norm_rotary_grad(dq, dk, q, k, wq, wk, positions, inv_freq, **how)
    assert all(a is b is None or torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("weights", ["both", "q", "k"])
def test_autograd(weights):
    """Gradients through autograd are the direct ones', whichever inputs ask for them, also of strided tensors."""
    import paged_cache as pc
    fused = _randn(1, (50, 6, 64), BF16)
    q, k = fused[:, :4], fused[:, 4:]
    wq = _randn(3, (64,), BF16) if weights != "k" else None
    wk = _randn(4, (64,), BF16) if weights != "q" else None
    positions, inv_freq = torch.arange(50, device=DEV), torch.rand(32, device=DEV)
    dq, dk = _randn(6, q.shape, BF16), torch.ones((), dtype=BF16, device=DEV).expand(k.shape)
    want = pc.norm_rotary_grad(dq, dk.contiguous(), q, k, wq, wk, positions, inv_freq)
    fused.requires_grad_()
    leaves = [fused] + [w.requires_grad_() for w in (wq, wk) if w is not None]
    y, z = pc.norm_rotary(fused[:, :4], fused[:, 4:], wq, wk, positions, inv_freq)
    got = torch.autograd.grad([y, z], leaves, [dq, dk])
    assert torch.equal(got[0], torch.cat(want[:2], dim=1))
    for g, w in zip(got[1:], [w for w in want[2:] if w is not None]):
        assert torch.equal(g, w)


def test_q_alone_and_inputs_as_outputs_of_nothing():
    import paged_cache as pc
    q, k, wq, wk, positions, inv_freq, sections = _setup(20, 3, 2, 64, (32,), F32, F32)
    y, none = pc.norm_rotary(q, None, wq, None, positions, inv_freq)
    assert none is None and torch.equal(y, pc.norm_rotary(q, k, wq, wk, positions, inv_freq)[0])
    dq = _randn(6, q.shape, F32)
    got = pc.norm_rotary_grad(dq, None, q, None, wq, None, positions, inv_freq)
    assert got[1] is None and got[3] is None
    assert torch.equal(got[0], pc.norm_rotary_grad(dq, dq[:, :2], q, k, wq, wk, positions, inv_freq)[0])


@pytest.mark.parametrize("T", [0, 1])
def test_no_tokens_and_one(T):
    import paged_cache as pc
    q, k, wq, wk, positions, inv_freq, _ = _setup(T, 3, 2, 64, (32,), BF16, BF16)
    y, z = pc.norm_rotary(q, k, wq, wk, positions, inv_freq)
    assert y.shape == q.shape and z.shape == k.shape
    got = pc.norm_rotary_grad(q, k, q, k, wq, wk, positions, inv_freq)
    if T == 0:
        assert torch.all(got[2] == 0) and torch.all(got[3] == 0)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("scale,eps", [(1e30, 1e-6), (1e-30, 1e-6), (1e-30, 0.0), (1e-3, 1e-6)])
def test_values_whose_squares_leave_the_range(scale, eps, dtype):
    import paged_cache as pc
    print(f"[case] norm rotary values of {scale} {eps} {dtype}", flush=True)
    q, k, wq, wk, positions, inv_freq, sections = _setup(12, 3, 2, 128, (64,), dtype, F32, scale)
    y, z = pc.norm_rotary(q, k, wq, wk, positions, inv_freq, eps=eps)
    args = (positions, inv_freq, sections, eps)
    _check("q", y, ref.forward(q, wq, *args))
    _check("k", z, ref.forward(k, wk, *args))
    if scale != 1e30 and eps:
        dq, dk = _randn(6, q.shape, dtype, 1e-3), _randn(7, k.shape, dtype, 1e-3)
        got = pc.norm_rotary_grad(dq, dk, q, k, wq, wk, positions, inv_freq, eps=eps)
        _check("dq", got[0], ref.gradients(dq, q, wq, *args)[0])


def test_rows_of_zeros_and_of_nan_touch_no_other():
    import paged_cache as pc
    q, k, wq, wk, positions, inv_freq, _ = _setup(9, 4, 2, 64, (32,), BF16, BF16)
    want, _ = pc.norm_rotary(q, k, wq, wk, positions, inv_freq)
    x = q.clone()
    x[2, 1], x[5, 3] = 0.0, float("nan")
    y, _ = pc.norm_rotary(x, k, wq, wk, positions, inv_freq)
    assert torch.all(y[2, 1] == 0) and torch.all(torch.isnan(y[5, 3]))
    y[2, 1], y[5, 3] = want[2, 1], want[5, 3]
    assert torch.equal(y, want)


def test_gradients_against_differences():
    """Difference quotients of sum(y dy) in fp32 over a step of 1e-2 times a unit direction: h^2 / 6 of a third derivative of
    order |dy| / rms^2 (rms near 1), and the sums' rounding over h."""
    import paged_cache as pc
    q, k, wq, wk, positions, inv_freq, _ = _setup(7, 2, 1, 64, (32,), F32, F32, 1.0)
    dy = _randn(8, q.shape, F32)
    zero = torch.zeros_like(k)
    got = pc.norm_rotary_grad(dy, zero, q, k, wq, wk, positions, inv_freq)

    def value(x, w):
        return (pc.norm_rotary(x, k, w, wk, positions, inv_freq)[0].double() * dy.double()).sum().item()
    h = 1e-2
    rounding = 64 * 2.0 ** -24 * dy.abs().sum().item() * 3 / h
    t = _randn(9, q.shape, F32)
    t /= t.norm()
    quotient = (value(q + h * t, wq) - value(q - h * t, wq)) / (2 * h)
    assert abs(quotient - (got[0].double() * t.double()).sum().item()) <= 4 * h ** 2 + rounding
    t = _randn(10, wq.shape, F32)
    t /= t.norm()
    quotient = (value(q, wq + h * t) - value(q, wq - h * t)) / (2 * h)
    assert abs(quotient - (got[2].double() * t.double()).sum().item()) <= rounding


def test_a_captured_step_replays():
    import paged_cache as pc
    q, k, wq, wk, positions, inv_freq, _ = _setup(90, 4, 2, 128, (64,), BF16, BF16)
    bufs = [q.clone(), k.clone()]

    def step(a, b):
        return (*pc.norm_rotary(a, b, wq, wk, positions, inv_freq),
                *pc.norm_rotary_grad(a, b, a, b, wq, wk, positions, inv_freq))
    step(*bufs)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step(*bufs)
    for rep in range(3):
        new = [_randn(50 + rep, x.shape, BF16) for x in bufs]
        for b, x in zip(bufs, new):
            b.copy_(x)
        want = step(*new)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), rep
