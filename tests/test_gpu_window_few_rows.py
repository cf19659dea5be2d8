"""GPU: the gradient of a few queries over many keys, in which fp16 has a pass over v that other types have not."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _time(call):
    """The fastest of five calls, ms."""
    call()
    best = float("inf")
    for _ in range(5):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        call()
        b.record()
        torch.cuda.synchronize()
        best = min(best, a.elapsed_time(b))
    return best


def test_one_query_over_many_keys_takes_fp16_no_longer_than_bf16():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    import window_attention as wa
    S, H, D = 1 << 17, 8, 64
    times = {}
    for dtype in (torch.bfloat16, torch.float16):
        g = torch.Generator(DEV).manual_seed(1)
        q, k, v, dout = (torch.randn((n, H, D), generator=g, device=DEV, dtype=dtype) for n in (1, S, S, 1))
        out, lse, rest = wa.window_attention(q, k, v, want_lse=True, want_rest=True)
        times[dtype] = _time(lambda: wa.window_attention_grad(dout, q, k, v, out, lse, rest))
    print(f"[case] one query over {S} keys: {times}", flush=True)
    # the pass over v reads half of what the others read; with one workgroup for all of v it took several times as long
    assert times[torch.float16] < 2 * times[torch.bfloat16], times
