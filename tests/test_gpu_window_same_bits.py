"""GPU: attention with a window gives the same bits whether a gradient is wanted or not, as a pass that is formed again
before its backward pass needs."""
import pytest
import torch
import torch.utils.checkpoint

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("H,D", [(2, 128), (40, 64)])
@pytest.mark.parametrize("T,window", [(200, None), (700, None), (1500, None), (1500, 400), (1500, 900)])
def test_with_and_without_gradients(T, window, H, D, dtype):
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    import window_attention as wa
    print(f"[case] window bits {T} {window} {H} {D} {dtype}", flush=True)
    g = torch.Generator().manual_seed(T)
    q, k, v = (torch.randn((T, H, D), generator=g).to(dtype).to(DEV) for _ in range(3))
    want, lse = wa.window_attention(q, k, v, window=window, sinks=2, want_lse=True)
    for _ in range(2):
        assert torch.equal(wa.window_attention(q, k, v, window=window, sinks=2), want)
    q.requires_grad_()
    out, lse2 = wa.window_attention(q, k, v, window=window, sinks=2, want_lse=True)
    assert out.requires_grad and torch.equal(out, want) and torch.equal(lse, lse2)
    with torch.no_grad():
        assert torch.equal(wa.window_attention(q, k, v, window=window, sinks=2, want_rest=True)[0], want)

    def layer(q):
        return wa.window_attention(q, k, v, window=window, sinks=2)
    plain, = torch.autograd.grad(layer(q), q, torch.ones_like(want))
    again = torch.utils.checkpoint.checkpoint(layer, q, use_reentrant=False)
    assert torch.equal(again, want) and torch.equal(torch.autograd.grad(again, q, torch.ones_like(want))[0], plain)
