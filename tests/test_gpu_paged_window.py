"""GPU: paged attention with a window and sinks, and behind a shared prefix, against the definitions in 64 bits, and runs
of the new operators together.

Tolerance, as for paged attention: a score is off by at most (D + 8) u S, u = 2^-24 and S = sm_scale max_j sum_d |q_d
k_jd|; p by twice that, its two parts by 2^-16, its sum over n keys by n + 64 roundings: out is off by at most
(2 (D + 8) u S + (n + 64) u + 2^-16) R with R = sum_j p_j |v_j|, plus half a step of its type."""
import pytest
import torch

import window_ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    import _sta_native
    _sta_native.lib()


def _randn(seed, shape, dtype, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(DEV)


def _paged(seed, lens, page, Hkv, D, dtype, extra=0):
    """Pages filled at random, NaN where no key is, and a table of them in a shuffled order; extra pages more, unused."""
    import paged_cache as pc
    need = [-(-n // page) for n in lens]
    pages = sum(need) + extra + 1
    ids = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(lens), max(max(need), 1)), -1, dtype=torch.int32)
    k = torch.full((pages, Hkv, page, D), float("nan"), dtype=dtype, device=DEV)
    v = k.clone()
    at = 0
    for b, n in enumerate(lens):
        for x in range(need[b]):
            p, m = ids[at], min(page, n - x * page)
            table[b, x] = p
            k[p, :, :m], v[p, :, :m] = _randn(seed + 2 * at + 1, (Hkv, m, D), dtype), _randn(seed + 2 * at + 2, (Hkv, m, D), dtype)
            at += 1
    return pc.PagedCache(k, v), table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), ids[at:at + extra]


def _keys(pages, row, n):
    page = pages.shape[2]
    j = torch.arange(n, device=DEV)
    p = row[j // page].long()
    there = p >= 0
    rows = pages[p.clamp(min=0), :, j % page].double().transpose(0, 1)            # (Hkv, n, D)
    return torch.where(there[None, :, None], rows, 0.0), there


def _check(q, cache, table, lens, got, lse, window=None, sinks=0, prefix=None, prefix_len=0):
    q4 = q if q.dim() == 4 else q[:, :, None]
    got, lse = (got if q.dim() == 4 else got[:, :, None]).double(), lse if q.dim() == 4 else lse[:, :, None]
    B, H, Q, D = q4.shape
    Hkv, e, scale = cache.kv_heads, torch.finfo(q.dtype).eps / 2, q.shape[-1] ** -0.5
    tiny = torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps
    for b, n in enumerate(lens):
        k, there = _keys(cache.k, table[b], n)
        v, _ = _keys(cache.v, table[b], n)
        sees = window_ref.visible(Q, n, window, sinks, DEV) & there
        if prefix is not None:
            kp, tp = _keys(cache.k, prefix, prefix_len)
            vp, _ = _keys(cache.v, prefix, prefix_len)
            k, v = torch.cat([kp, k], dim=1), torch.cat([vp, v], dim=1)
            sees = torch.cat([tp.expand(Q, -1), sees], dim=1)
        some, m = sees.any(dim=1), k.shape[1]
        for h in range(H):
            kh, vh, qh = k[h // (H // Hkv)], v[h // (H // Hkv)], q4[b, h].double()
            s = (qh @ kh.t() * scale).masked_fill(~sees, float("-inf"))
            l = torch.logsumexp(s, dim=1)
            p = torch.exp(s - torch.where(some, l, 0.0)[:, None]).masked_fill(~sees, 0.0)
            S = (qh.abs() @ kh.abs().t() * scale).masked_fill(~sees, 0.0).amax(dim=1) if m else torch.zeros(Q, device=DEV)
            rp = (2 * (D + 8) * S + m + 64) * U
            want, R = p @ vh, p @ vh.abs()
            bound = (rp[:, None] + 2.0 ** -16) * R + e * want.abs() + tiny
            err = (got[b, h] - want).abs()
            assert torch.all(err <= bound), f"sequence {b} head {h}: {(err - bound).max().item():.3e} beyond the bound"
            assert torch.equal(lse[b, h] == float("-inf"), ~some)
            assert torch.all(((lse[b, h].double() - l).abs() <= rp + 8 * U * (l.abs() + 1)) | ~some)


@pytest.mark.parametrize("dtype,H,Hkv,D", [(BF16, 8, 2, 128), (F16, 4, 4, 64), (F32, 6, 2, 128), (BF16, 40, 1, 64)])
@pytest.mark.parametrize("Q,page", [(1, 16), (1, 1), (2, 8), (5, 32), (33, 64), (40, 4)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (7, 4), (100, 0), (64, 9), (500, 130), (3000, 3)])
def test_window(window, sinks, Q, page, dtype, H, Hkv, D):
    import paged_cache as pc
    if page == 1 and window > 100:
        pytest.skip("the same walk as larger pages")
    lens = [1, 0, 700, 64, 2049, 100, 33]
    if page == 1:
        lens = [1, 0, 130, 64]
    print(f"[case] paged window {window} {sinks} Q={Q} page={page} {dtype} {H} {Hkv} {D}", flush=True)
    cache, table, d_lens, _ = _paged(7, lens, page, Hkv, D, dtype)
    q = _randn(3, (len(lens), H, D) if Q == 1 else (len(lens), H, Q, D), dtype, 2.0)
    out, lse = pc.paged_attention(q, cache, table, d_lens, want_lse=True, window=window, sinks=sinks)
    _check(q, cache, table, lens, out, lse, window, sinks)


def test_a_window_that_reaches_every_key_is_none():
    import paged_cache as pc
    cache, table, lens, _ = _paged(1, [300, 20, 5], 16, 2, 64, BF16)
    q = _randn(3, (3, 8, 64), BF16)
    want = pc.paged_attention(q, cache, table, lens)
    assert torch.equal(pc.paged_attention(q, cache, table, lens, window=304, sinks=2), want)
    assert torch.equal(pc.paged_attention(q, cache, table, lens, window=2 ** 40, sinks=2 ** 40), want)


@pytest.mark.parametrize("Q", [1, 3])
def test_pages_that_left_the_window_may_be_gone(Q):
    import paged_cache as pc
    lens = [900, 411, 37]
    cache, table, d_lens, _ = _paged(5, lens, 16, 2, 128, BF16)
    q = _randn(3, (3, 4, Q, 128), BF16)
    want = pc.paged_attention(q, cache, table, d_lens, window=100, sinks=20)
    gone = table.clone()
    for b, n in enumerate(lens):
        first = max(n - (Q - 1) - 100, 0) // 16
        gone[b, 2:max(first, 2)] = -1
    assert (gone != table).any()
    assert torch.equal(pc.paged_attention(q, cache, gone, d_lens, window=100, sinks=20), want)


def test_keys_outside_the_window_reach_nothing():
    """NaN and infinities in front of the window, between the sinks and it, and in its edge pages."""
    import paged_cache as pc
    for Q in (1, 4, 40):
        cache, table, lens, _ = _paged(9, [500, 500], 32, 2, 64, BF16)
        q = _randn(3, (2, 8, Q, 64), BF16)
        want = pc.paged_attention(q, cache, table, lens, window=70, sinks=5)
        j = torch.arange(5, 500 - (Q - 1) - 70, device=DEV)
        for pages, bad in ((cache.k, float("nan")), (cache.v, float("inf"))):
            pages[table[0, j // 32].long(), :, j % 32] = bad
        assert torch.equal(pc.paged_attention(q, cache, table, lens, window=70, sinks=5), want), Q


@pytest.mark.parametrize("dtype,H,Hkv,D", [(BF16, 8, 2, 128), (F16, 4, 4, 64), (F32, 6, 2, 128), (BF16, 40, 1, 64)])
@pytest.mark.parametrize("Q,page", [(1, 16), (1, 4), (2, 8), (5, 64)])
@pytest.mark.parametrize("prefix_len,lens", [(1, [0, 1, 40]), (33, [5, 0, 300, 2, 7, 1, 64, 90, 11, 3]), (2500, [10, 700, 0]),
                                             (640, [1])])
def test_prefix(prefix_len, lens, Q, page, dtype, H, Hkv, D):
    import paged_cache as pc
    print(f"[case] prefix {prefix_len} {lens} Q={Q} page={page} {dtype} {H} {Hkv} {D}", flush=True)
    cache, table, d_lens, _ = _paged(11, [prefix_len, *lens], page, Hkv, D, dtype)
    prefix, own = table[0], table[1:]
    q = _randn(3, (len(lens), H, D) if Q == 1 else (len(lens), H, Q, D), dtype, 2.0)
    out, lse = pc.prefix_attention(q, cache, prefix, prefix_len, own, d_lens[1:], want_lse=True)
    _check(q, cache, own, lens, out, lse, prefix=prefix, prefix_len=prefix_len)


def test_prefix_with_lost_pages_many_rows_and_strides():
    """Prefix pages without an entry count as no keys; queries whose batch stride is not their queries' together; 300 rows
    and more a kv head."""
    import paged_cache as pc
    lens = [20, 3, 0, 77, 50, 9, 31, 200, 15, 64]
    cache, table, d_lens, _ = _paged(13, [1000, *lens], 16, 2, 128, BF16)
    prefix = table[0].clone()
    prefix[3], prefix[40] = -1, -1
    q = _randn(3, (8, 10, 9, 128), BF16, 2.0).permute(1, 0, 2, 3)[:, :, 1:6]
    out, lse = pc.prefix_attention(q, cache, prefix, 1000, table[1:], d_lens[1:], want_lse=True)
    _check(q, cache, table[1:], lens, out, lse, prefix=prefix, prefix_len=1000)
    # all of it gone: the own keys alone
    alone = pc.prefix_attention(q, cache, torch.full_like(prefix, -1), 1000, table[1:], d_lens[1:])
    want = pc.paged_attention(q, cache, table[1:], d_lens[1:])
    assert (alone.double() - want.double()).abs().max() <= 4 * torch.finfo(BF16).eps * want.abs().max()


def test_large_values_in_prefix_and_own_keys():
    """Sums of values near the type's largest do not pass it when both parts are joined."""
    import paged_cache as pc
    lens = [90, 0, 300]
    cache, table, d_lens, _ = _paged(15, [400, *lens], 16, 1, 64, F32)
    cache.v.copy_(torch.where(torch.isnan(cache.v), cache.v, 3e38))
    q = torch.zeros((3, 2, 64), device=DEV)
    out = pc.prefix_attention(q, cache, table[0], 400, table[1:], d_lens[1:])
    assert torch.all((out / 3e38 - 1).abs() <= 700 * 2.0 ** -24)


def test_a_serving_step_and_its_graph():
    """Norm and rotation, append, attention behind a prefix in one layer and with a window in the next: against the same
    step over one contiguous text, and replayed from a graph."""
    import paged_cache as pc
    B, H, Hkv, D, page, n0, W = 5, 8, 2, 64, 16, 150, 60
    own = [33, 0, 80, 5, 64]
    cache, table, d_lens, _ = _paged(17, [n0, *[n + 1 for n in own]], page, Hkv, D, BF16)
    prefix, table = table[0], table[1:].contiguous()
    flat = torch.cat([prefix.expand(B, -1), table], dim=1).contiguous()
    lens = torch.tensor(own, dtype=torch.int32, device=DEV)
    wq, wk = 1 + _randn(1, (D,), BF16, 0.2), 1 + _randn(2, (D,), BF16, 0.2)
    inv_freq = (1e4 ** -(torch.arange(D // 2) / (D // 2))).to(DEV)
    xs = [_randn(3, (B, H, D), BF16), _randn(4, (B, Hkv, D), BF16), _randn(5, (B, Hkv, D), BF16)]

    def step(q, k, v):
        q, k = pc.norm_rotary(q, k, wq, wk, lens + n0, inv_freq)
        grown = pc.cache_append(cache, k, v, table, lens)
        far = pc.prefix_attention(q, cache, prefix, n0, table, grown, max_len=96)
        near = pc.paged_attention(q, cache, table, grown, max_len=96, window=W, sinks=4)
        return q, far, near, grown
    q, far, near, grown = step(*xs)
    for b, n in enumerate(own):
        k, _ = _keys(cache.k, torch.cat([prefix, table[b]]), flat.shape[1] * page)
        v, _ = _keys(cache.v, torch.cat([prefix, table[b]]), flat.shape[1] * page)
        at = torch.cat([torch.arange(n0), prefix.shape[0] * page + torch.arange(n + 1)]).to(DEV)
        r = window_ref.attention(q[b:b + 1], k[:, at].transpose(0, 1), v[:, at].transpose(0, 1), None, 0, None, None, D ** -0.5)
        assert torch.all((far[b:b + 1].double() - r["out"][0]).abs() <= r["out"][1])
        at = at[n0:]
        r = window_ref.attention(q[b:b + 1], k[:, at].transpose(0, 1), v[:, at].transpose(0, 1), W, 4, None, None, D ** -0.5)
        assert torch.all((near[b:b + 1].double() - r["out"][0]).abs() <= r["out"][1])
    bufs = [x.clone() for x in xs]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step(*bufs)
    for rep in range(3):
        new = [_randn(30 + 3 * rep + i, x.shape, BF16) for i, x in enumerate(xs)]
        for b, x in zip(bufs, new):
            b.copy_(x)
        want = [x.clone() for x in step(*new)]
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), rep


def test_a_window_layer_trains_packed_and_serves_paged():
    """The same tokens through window_attention as packed sequences and, the last ones, through the paged cache."""
    import paged_cache as pc
    import window_attention as wa
    lens, H, Hkv, D, Q, page = [70, 9, 150], 4, 2, 64, 3, 16
    T = sum(lens)
    starts = torch.tensor([0, 70, 79, 229], dtype=torch.int32, device=DEV)
    x = [_randn(i, (T, h, D), BF16) for i, h in enumerate([H, Hkv, Hkv])]
    wq, wk = 1 + _randn(8, (D,), BF16, 0.2), 1 + _randn(9, (D,), BF16, 0.2)
    positions = torch.cat([torch.arange(n) for n in lens]).to(DEV)
    inv_freq = (1e4 ** -(torch.arange(D // 2) / (D // 2))).to(DEV)
    leaves = [y.requires_grad_() for y in (*x, wq, wk)]
    q, k = pc.norm_rotary(x[0], x[1], wq, wk, positions, inv_freq)
    out = wa.window_attention(q, k, x[2], window=40, sinks=2, starts=starts)
    grads = torch.autograd.grad(out.float().square().sum(), leaves)
    assert all(torch.isfinite(g).all() and g.abs().max() > 0 for g in grads)
    q, k, v, out = q.detach(), k.detach(), x[2].detach(), out.detach()
    table = torch.arange(30, dtype=torch.int32, device=DEV).view(3, 10)
    cache = pc.PagedCache.empty(30, page, Hkv, D, evictable=False)
    grown = pc.cache_append(cache, k, v, table, torch.zeros(3, dtype=torch.int32, device=DEV), starts)
    last = torch.stack([torch.arange(e - Q, e) for e in (70, 79, 229)]).to(DEV)
    served = pc.paged_attention(q[last].transpose(1, 2), cache, table, grown, window=40, sinks=2).transpose(1, 2)
    want = window_ref.attention(q, k, v, 40, 2, starts.tolist(), None, D ** -0.5)["out"]
    assert torch.all((served.double() - want[0][last]).abs() <= want[1][last])
    assert torch.all((out.double() - want[0]).abs() <= want[1])
