"""CPU checks of how rotary takes part in automatic differentiation, with the formula in place of the launch."""
import pytest
import torch
import torch.autograd.forward_ad as fwad


def _formula(q, k, positions, inv_freq, sections=None, pos_scale=1.0, rope_scale=1.0, inverse=False):
    half = inv_freq.numel()
    axis = [a for a, n in enumerate(sections or (half,)) for _ in range(n)]
    angle = positions.reshape(-1, positions.shape[-1])[axis].t() * pos_scale * inv_freq           # (T, half)
    c, s = angle.cos()[:, None] * rope_scale, angle.sin()[:, None] * (-rope_scale if inverse else rope_scale)

    def turn(x):
        assert type(x) is torch.Tensor and fwad.unpack_dual(x).tangent is None, "the launch takes plain tensors"
        a, b = x[..., :half], x[..., half:2 * half]
        return torch.cat([a * c - b * s, b * c + a * s, x[..., 2 * half:]], dim=-1)
    return turn(q), None if k is None else turn(k)


@pytest.fixture
def pc(monkeypatch):
    import paged_cache
    monkeypatch.setattr(paged_cache.native, "rotary", _formula)
    return paged_cache


HOW = ((8, 8), 0.5, 1.25)
# products and sums of the same numbers in another order: a few steps of 2^-53
CLOSE = dict(rtol=0, atol=64 * 2.0 ** -53)


def _made():
    g = torch.Generator().manual_seed(1)
    q, k, tq, tk = (torch.randn((5, h, 40), generator=g, dtype=torch.float64) for h in (3, 2, 3, 2))
    return q, k, tq, tk, torch.arange(10.0, dtype=torch.float64).reshape(2, 5), torch.rand(16, generator=g).double()


@pytest.mark.parametrize("no_grad", [False, True])
@pytest.mark.parametrize("which", ["q", "k", "both", "q alone"])
def test_forward_mode_carries_the_tangents(pc, which, no_grad):
    """The rotation is linear in q and k: its tangents are their tangents, rotated."""
    q, k, tq, tk, pos, inv = _made()
    with torch.autograd.grad_mode.set_grad_enabled(not no_grad), fwad.dual_level():
        dual_q = fwad.make_dual(q, tq) if which != "k" else q
        dual_k = None if which == "q alone" else fwad.make_dual(k, tk) if which != "q" else k
        a, b = pc.rotary(dual_q, dual_k, pos, inv, *HOW)
        want = _formula(tq if which != "k" else torch.zeros_like(q), tk if which in ("k", "both") else torch.zeros_like(k),
                        pos, inv, *HOW)
        for got, x, t in ((a, q, want[0]), (b, k, want[1])):
            if got is None:
                assert which == "q alone"
                continue
            p = fwad.unpack_dual(got)
            tangent = torch.zeros_like(x) if p.tangent is None else p.tangent
            torch.testing.assert_close(tangent, t, **CLOSE)
        torch.testing.assert_close(fwad.unpack_dual(a).primal, _formula(q, None, pos, inv, *HOW)[0], **CLOSE)


def test_forward_over_reverse_and_function_transforms(pc):
    q, k, tq, tk, pos, inv = _made()

    def loss(x):                                              # quadratic, so that its gradient has a derivative
        a, b = pc.rotary(x, k, pos, inv, *HOW)
        return (a * a * tq).sum() + (b * tk).sum()
    x = q.clone().requires_grad_()
    g, = torch.autograd.grad(loss(x), x)
    want = _formula(2 * tq * _formula(q, None, pos, inv, *HOW)[0], None, pos, inv, *HOW, inverse=True)[0]
    torch.testing.assert_close(g, want, **CLOSE)
    torch.testing.assert_close(torch.func.grad(loss)(q), want, **CLOSE)
    value, slope = torch.func.jvp(loss, (q,), (tq,))
    torch.testing.assert_close(slope, (want * tq).sum(), rtol=1e-12, atol=0)
    torch.testing.assert_close(value, loss(q), rtol=1e-12, atol=0)
    # the derivative of the gradient along tq
    hess = _formula(2 * tq * _formula(tq, None, pos, inv, *HOW)[0], None, pos, inv, *HOW, inverse=True)[0]
    with fwad.dual_level():
        d = fwad.make_dual(q.clone().requires_grad_(), tq)
        g, = torch.autograd.grad(loss(d), d, create_graph=True)
        torch.testing.assert_close(fwad.unpack_dual(g).tangent, hess, **CLOSE)
    torch.testing.assert_close(torch.func.jvp(torch.func.grad(loss), (q,), (tq,))[1], hess, **CLOSE)
    assert torch.autograd.gradcheck(lambda u, w: pc.rotary(u, w, pos, inv, *HOW), (q.clone().requires_grad_(),
                                    k.clone().requires_grad_()), check_forward_ad=True, check_backward_ad=True)


def test_plain_calls_stay_off_the_graph(pc):
    q, k, _, _, pos, inv = _made()
    a, b = pc.rotary(q, k, pos, inv, *HOW)
    assert a.grad_fn is None and b.grad_fn is None
    with torch.no_grad():
        a, _ = pc.rotary(q.clone().requires_grad_(), k, pos, inv, *HOW)
    assert a.grad_fn is None and not a.requires_grad


def test_the_raw_gradient_refuses_what_it_would_lose(pc):
    """rotary_grad is outside every graph: a tangent on its inputs raises instead of reading as zero."""
    q, k, tq, tk, pos, inv = _made()
    with fwad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            pc.rotary_grad(fwad.make_dual(q, tq), k, pos, inv, *HOW)
        with pytest.raises(RuntimeError, match="forward-mode"):
            pc.rotary_grad(q, fwad.make_dual(k, tk), pos, inv, *HOW)
        a, b = pc.rotary_grad(q, k, pos, inv, *HOW)
        torch.testing.assert_close(a, _formula(q, None, pos, inv, *HOW, inverse=True)[0], **CLOSE)
