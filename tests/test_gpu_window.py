"""GPU: attention over packed sequences with a sliding window and sinks, and its gradients, against the definitions
in 64 bits with the bounds derived in window_ref.py."""
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


def _starts(lens, first=0):
    s = [first]
    for n in lens:
        s.append(s[-1] + n)
    return torch.tensor(s, dtype=torch.int32, device=DEV)


def _check(name, got, want, bound):
    err = (got.double() - want).abs()
    same = (got.double() == want) | (torch.isnan(got.double()) & torch.isnan(want))    # infinities
    bad = ~(err <= bound) & ~same
    assert not bad.any(), (f"{name} off by {err[bad].max().item():.3e}, bound {bound[bad].max().item():.3e}, at "
                           f"{bad.nonzero()[0].tolist()}, {int(bad.sum())} of {bad.numel()}")


def _run(q, k, v, dout, window, sinks, starts, k_starts, sm_scale):
    import window_attention as wa
    q, k, v = (x.detach().requires_grad_() for x in (q, k, v))
    out, lse = wa.window_attention(q, k, v, window=window, sinks=sinks, starts=starts, k_starts=k_starts,
                                   sm_scale=sm_scale, want_lse=True)
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), dout)
    return {"out": out.detach(), "lse": lse, "dq": dq, "dk": dk, "dv": dv}


def _compare(q, k, v, dout, window, sinks, starts=None, k_starts=None, sm_scale=None):
    scale = q.shape[-1] ** -0.5 if sm_scale is None else sm_scale
    got = _run(q, k, v, dout, window, sinks, starts, k_starts, sm_scale)
    want = ref.attention(q, k, v, window, sinks, None if starts is None else starts.tolist(),
                         None if k_starts is None else k_starts.tolist(), scale, dout)
    for name, (value, bound) in want.items():
        _check(name, got[name], value, bound)
    return got


# (lengths of the sequences, window, sinks)
PACKED = [([1], None, 0), ([1, 1, 2], 1, 0), ([5, 0, 37, 1, 64], 3, 4), ([129, 33], 1, 1), ([257], 64, 0), ([300, 20], None, 0),
          ([31, 32, 33, 127, 128, 129], 40, 2), ([500], 100, 130), ([200, 190], 1000, 5), ([640], 33, 300)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("H,Hkv,D", [(4, 1, 128), (2, 2, 64)])
@pytest.mark.parametrize("lens,window,sinks", PACKED)
def test_packed_sequences(lens, window, sinks, H, Hkv, D, dtype):
    print(f"[case] window {lens} {window} {sinks} {H} {Hkv} {D} {dtype}", flush=True)
    T = sum(lens)
    q, k, v, dout = (_randn(i, (T, h, D), dtype, s) for i, (h, s) in enumerate([(H, 2.0), (Hkv, 1.0), (Hkv, 1.0), (H, 1.0)]))
    _compare(q, k, v, dout, window, sinks, _starts(lens))


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (F16, 64), (F32, 128), (F32, 64)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (700, 3), (90, 200)])
def test_workgroups_of_four_waves(window, sinks, dtype, D):
    """Enough rows for 128 a workgroup in both passes (300 and more of them)."""
    print(f"[case] window four waves {window} {sinks} {dtype} {D}", flush=True)
    lens = [1500, 1, 640, 0, 499]
    T, H, Hkv = sum(lens), 26, 13
    q, k, v, dout = (_randn(i, (T, h, D), dtype, s) for i, (h, s) in enumerate([(H, 2.0), (Hkv, 1.0), (Hkv, 1.0), (H, 1.0)]))
    _compare(q, k, v, dout, window, sinks, _starts(lens))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("window,sinks", [(None, 0), (50, 3)])
def test_rows_and_keys_of_different_counts(window, sinks, dtype):
    """Fewer queries than keys (a prompt behind cached keys), more (the first rows see nothing), none of one of them, and
    rows and keys in front of the first sequence and behind the last."""
    print(f"[case] window counts {window} {sinks} {dtype}", flush=True)
    nq, nk = [7, 40, 0, 1, 90, 13], [300, 40, 12, 77, 20, 0]
    starts, k_starts = _starts(nq, 5), _starts(nk, 9)
    T, S, H, Hkv, D = int(starts[-1]) + 21, int(k_starts[-1]) + 40, 4, 2, 64
    q, k, v, dout = _randn(1, (T, H, D), dtype, 2.0), _randn(2, (S, Hkv, D), dtype), _randn(3, (S, Hkv, D), dtype), \
        _randn(4, (T, H, D), dtype)
    outside = [torch.ones(n, dtype=torch.bool, device=DEV) for n in (T, S)]
    outside[0][5:-21] = outside[1][9:-40] = False
    for x, rows in ((q, 0), (dout, 0), (k, 1), (v, 1)):    # not read
        x[outside[rows]] = float("nan")
    got = _compare(q, k, v, dout, window, sinks, starts, k_starts)
    for name, rows in (("out", 0), ("dq", 0), ("dk", 1), ("dv", 1)):
        assert torch.all(got[name][outside[rows]] == 0), name
    assert torch.all(got["lse"][outside[0]] == float("-inf"))
    assert torch.all(got["out"][starts[4]:starts[4] + 70] == 0)          # 90 rows behind 20 keys: 70 see nothing


def test_one_sequence_without_starts_and_other_position_types():
    q, k, v, dout = (_randn(i, (150, 2, 64), BF16) for i in range(4))
    a = _compare(q, k, v, dout, 20, 2)
    b = _run(q, k, v, dout, 20, 2, torch.tensor([0, 150], device=DEV), None, None)      # int64
    for name in a:
        assert torch.equal(a[name], b[name]), name


@pytest.mark.parametrize("T,S", [(0, 0), (0, 30), (12, 0)])
def test_empty_tensors(T, S):
    q, k, v = _randn(1, (T, 2, 64), F16), _randn(2, (S, 2, 64), F16), _randn(3, (S, 2, 64), F16)
    got = _run(q, k, v, _randn(4, (T, 2, 64), F16), 4, 1, None, None, None)
    for name in ("out", "dq", "dk", "dv"):
        assert torch.all(got[name] == 0), name
    assert torch.all(got["lse"] == float("-inf"))


@pytest.mark.parametrize("sm_scale", [0.0, -0.2, 1.7, 1e-40])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_scales(sm_scale, dtype):
    print(f"[case] window scale {sm_scale} {dtype}", flush=True)
    q, k, v, dout = (_randn(i, (140, 2, 64), dtype) for i in range(4))
    _compare(q, k, v, dout, 30, 2, sm_scale=sm_scale)


def test_strides_and_expanded_gradients():
    """Heads first, a slice of a fused projection, values shared by the heads, and a gradient of stride 0."""
    g = _randn(1, (3, 8, 90, 64), BF16)
    q, k = g[0, :4].transpose(0, 1), g[1, :2].transpose(0, 1)
    v = _randn(2, (90, 1, 192), BF16)[:, :, 64:128].expand(90, 2, 64)
    want = _run(q.contiguous(), k.contiguous(), v.contiguous(), torch.ones((90, 4, 64), dtype=BF16, device=DEV), 25, 1, None,
                None, None)
    got = _run(q, k, v, torch.ones((), dtype=BF16, device=DEV).expand(90, 4, 64), 25, 1, None, None, None)
    for name in want:
        assert torch.equal(got[name], want[name]), name


def test_small_and_large_gradients_of_fp16():
    """fp16 holds neither the smallest nor the largest scores' gradients: their common scale is taken out."""
    q, k, v = (_randn(i, (200, 2, 128), F16) for i in range(3))
    for size in (6e-5, 2000.0):
        print(f"[case] window fp16 gradients of {size}", flush=True)
        _compare(q, k, v, _randn(4, (200, 2, 128), F16, size), None, 0)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_scores_of_minus_infinity_and_large_ones(dtype):
    """A row whose scores are all -inf gets zeros, as one that sees nothing; scores of some thousands stay exact."""
    q, k, v, dout = (_randn(i, (70, 1, 64), dtype) for i in range(4))
    q[:, :, 0], k[:, :, 0] = 1.0, float("-inf")
    got = _run(q, k, v, dout, None, 0, None, None, 0.125)
    assert torch.all(got["out"] == 0) and torch.all(got["lse"] == float("-inf")) and torch.all(got["dv"] == 0)
    q, k = _randn(5, (70, 1, 64), dtype, 20.0), _randn(6, (70, 1, 64), dtype, 20.0)
    _compare(q, k, v, dout, 32, 1)


def test_the_gradient_on_its_own_is_autograds_and_repeats_its_bits():
    import window_attention as wa
    starts = _starts([300, 80])
    q, k, v, dout = (_randn(i, (380, h, 128), BF16) for i, h in enumerate([8, 2, 2, 8]))
    want = _run(q, k, v, dout, 64, 3, starts, None, None)
    out, lse, rest = wa.window_attention(q, k, v, window=64, sinks=3, starts=starts, want_lse=True, want_rest=True)
    assert torch.equal(out, want["out"]) and torch.equal(lse, want["lse"])
    # out and what its rounding left are the result to 16 bits more
    exact = ref.attention(q, k, v, 64, 3, starts.tolist(), None, 128 ** -0.5)["out"][0]
    assert (out.double() + rest.double() - exact).abs().sum() < (out.double() - exact).abs().sum()
    for _ in range(3):
        grads = wa.window_attention_grad(dout, q, k, v, out, lse, rest, window=64, sinks=3, starts=starts)
        for name, x in zip(("dq", "dk", "dv"), grads):
            assert torch.equal(x, want[name]), name
    without = wa.window_attention_grad(dout, q, k, v, out, lse, window=64, sinks=3, starts=starts)
    assert torch.equal(without[2], want["dv"])


def test_gradients_against_differences():
    """The change of sum(out dout) along a direction, in fp32, against the gradient's: the difference quotient over a step h is
    off by h^2 / 6 of a third derivative (h 1e-2, derivatives near 1 in each of the terms' few units) and by 2 u sum|out dout| / h."""
    import window_attention as wa
    starts = _starts([40, 23])
    x = [_randn(i, (63, h, 64), F32, 0.5) for i, h in enumerate([2, 1, 1])]
    dout, step = _randn(5, (63, 2, 64), F32), 1e-2
    got = _run(*x, dout, 9, 2, starts, None, None)

    def value(*y):
        return (wa.window_attention(*y, window=9, sinks=2, starts=starts).double() * dout.double()).sum().item()
    for i, name in enumerate(("dq", "dk", "dv")):
        t = _randn(10 + i, x[i].shape, F32)
        t /= t.norm()
        up, down = ([*x[:i], x[i] + sign * step * t, *x[i + 1:]] for sign in (1, -1))
        quotient = (value(*up) - value(*down)) / (2 * step)
        rounding = 64 * 2.0 ** -24 * (got["out"] * dout).abs().sum().item() / step
        assert abs(quotient - (got[name].double() * t.double()).sum().item()) <= step ** 2 + rounding, name


def test_a_captured_training_step_replays():
    """Forward and gradient in a graph, replayed on new inputs in place, with eager calls and an eager graph's backward
    between the replays."""
    import window_attention as wa
    starts = _starts([200, 60])
    ins = [_randn(i, (260, h, 64), BF16) for i, h in enumerate([4, 2, 2, 4])]
    bufs = [x.clone() for x in ins]

    def step(q, k, v, dout):
        out, lse, rest = wa.window_attention(q, k, v, window=50, sinks=2, starts=starts, want_lse=True, want_rest=True)
        return (out, *wa.window_attention_grad(dout, q, k, v, out, lse, rest, window=50, sinks=2, starts=starts))
    step(*bufs)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step(*bufs)
    for rep in range(4):
        new = [_randn(100 + 10 * rep + i, x.shape, BF16) for i, x in enumerate(ins)]
        for b, x in zip(bufs, new):
            b.copy_(x)
        eager = _run(*new, 50, 2, starts, None, None)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for x, name in zip(got, ("out", "dq", "dk", "dv")):
            assert torch.equal(x, eager[name]), f"replay {rep}: {name}"


def test_another_stream():
    q, k, v, dout = (_randn(i, (300, 4, 128), F16) for i in range(4))
    want = _run(q, k, v, dout, 77, 1, None, None, None)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = _run(q, k, v, dout, 77, 1, None, None, None)
    s.synchronize()
    for name in want:
        assert torch.equal(got[name], want[name]), name


def test_many_sequences():
    """More sequences than lanes, so that the search for a tile's takes several turns."""
    g = torch.Generator().manual_seed(3)
    lens = torch.randint(0, 9, (200,), generator=g).tolist()
    T = sum(lens)
    q, k, v, dout = (_randn(i, (T, 2, 64), BF16) for i in range(4))
    _compare(q, k, v, dout, 4, 1, _starts(lens))
