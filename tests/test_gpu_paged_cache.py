"""GPU: rotary positions, the paged cache, attention over it and eviction, against their definitions in
64 bits (paged_ref.py).

Tolerances.  u = 2^-24 is half a step of fp32, e = finfo.eps / 2 half a step of the output's type.
Rotation: the sine and cosine of an angle reduced in 64 bits are off by at most 4 u (the fraction of a turn
rounds to u / 2 of up to 1, times pi, and two steps of the function), the products and their difference
round three times: (8 u) (|x| + |y|) scale, plus e |out|.
Attention: a score is a sum of D products in fp32, off by at most (D + 8) u S with S = sm_scale max_j sum_d
|q_d k_jd| (the 8: the scale, the exponent's argument); p then carries a factor within 2 (D + 8) u S
of 1, its sum and the sum over n keys n + 64 roundings: out is off by at most (2 (D + 8) u S + (n + 64) u) R
with R = sum_j p_j |v_j|, plus e |out|; a weight by the same factor of the weight plus its own row sums.
"""
import math

import pytest
import torch

import paged_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
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


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


# -------------------------------------------------------------------------------------------- rotary
def _check_rotary(x, got, positions, inv_freq, sections, pos_scale=1.0, rope_scale=1.0, inverse=False):
    want, size = ref.rotary(x, positions, inv_freq, sections, pos_scale, rope_scale, inverse)
    # behind the rotated part size is 0: those elements are copies
    tiny = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps     # a step of the subnormal range
    tol = torch.where(size > 0, 8 * U * size + _half_step(x.dtype) * want.abs() * 1.001 + tiny, 0.0)
    err = (got.double().cpu() - want).abs()
    assert torch.all(err <= tol), f"off by {(err - tol).max().item():.3e} beyond the bound"


@pytest.mark.parametrize("T,H,Hkv,D,sections,dtype", [
    (1, 8, 2, 128, (64,), BF16), (37, 5, 1, 128, (16, 24, 24), BF16), (300, 4, 4, 64, (32,), F16),
    (65, 3, 3, 80, (8, 16, 16), F32), (7, 2, 1, 128, (16, 8, 8), BF16), (1025, 2, 2, 64, (8, 24), F32),
    (33, 1, 7, 16, (8,), F16), (9, 40, 8, 128, (1, 2, 3, 58), BF16), (5, 2, 2, 512, (256,), F32),
    (2100, 3, 1, 24, (8,), BF16)])
def test_rotary_and_its_gradient(T, H, Hkv, D, sections, dtype):
    import paged_cache as pc
    print(f"[case] rotary T={T} H={H} Hkv={Hkv} D={D} {sections} {dtype}", flush=True)
    half = sum(sections)
    q, k = _randn(1, (T, H, D), dtype), _randn(2, (T, Hkv, D), dtype)
    inv_freq = (10000.0 ** -(torch.arange(half, dtype=torch.float64) / half)).float().to(DEV)
    positions = torch.randint(0, 1 << 20, (len(sections), T), generator=torch.Generator().manual_seed(3),
                              dtype=torch.int32).to(DEV)
    a, b = pc.rotary(q, k, positions, inv_freq, sections)
    _check_rotary(q, a, positions, inv_freq, sections)
    _check_rotary(k, b, positions, inv_freq, sections)
    a, b = pc.rotary_grad(q, k, positions, inv_freq, sections, 0.25, 1.5)
    _check_rotary(q, a, positions, inv_freq, sections, 0.25, 1.5, True)
    _check_rotary(k, b, positions, inv_freq, sections, 0.25, 1.5, True)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64, torch.float32])
def test_rotary_position_types_strides_and_one_input(dtype):
    import paged_cache as pc
    x = _randn(4, (6, 21, 2, 64), BF16)
    q = x[3].transpose(0, 1).transpose(0, 1)[:, :1]           # strided tokens
    heads_first = _randn(5, (4, 21, 64), BF16).transpose(0, 1)
    inv_freq = torch.rand(32, generator=torch.Generator().manual_seed(6)).to(DEV)
    base = torch.arange(42, device=DEV) * 997 - 2000
    positions = (base.to(dtype) + (0.25 if dtype == torch.float32 else 0)).reshape(21, 2).t()   # strided, negative too
    got, none = pc.rotary(q, None, positions, inv_freq, (8, 24))
    assert none is None
    _check_rotary(q, got, positions, inv_freq, (8, 24))
    got, again = pc.rotary(heads_first, q, positions[1], inv_freq)
    _check_rotary(heads_first, got, positions[1:], inv_freq, (32,))
    _check_rotary(q, again, positions[1:], inv_freq, (32,))
    odd = _randn(7, (9, 3, 67), F32)[..., 1:65]               # rows that are not 16-byte aligned
    got, _ = pc.rotary(odd, None, positions[0, :9], inv_freq)
    _check_rotary(odd, got, positions[:1, :9], inv_freq, (32,))
    empty, none = pc.rotary(q[:0], None, positions[0, :0], inv_freq)
    assert empty.shape == (0, 1, 64)


def test_rows_that_begin_anywhere_and_dims_of_size_one():
    """Tensors that count as contiguous and whose address or strides are no multiples of 16 bytes."""
    import paged_cache as pc
    inv = (10000.0 ** -(torch.arange(64) / 64.0)).to(DEV)
    flat = _randn(5, (4 * 2 * 128 + 1,), BF16)
    shifted = flat[1:].view(4, 2, 128)                       # 2 bytes behind an aligned address
    single = _randn(6, (3, 2 * 128 + 4), BF16)[1:2, :256].unflatten(1, (2, 128))     # one token, rows of 260 elements
    pos4, pos1 = torch.arange(4, device=DEV), torch.arange(1, device=DEV) + 9
    for x, pos in ((shifted, pos4), (single, pos1)):
        assert x.is_contiguous()
        y, none = pc.rotary(x, None, pos, inv)
        assert none is None
        _check_rotary(x, y, pos[None], inv, (64,))
    made = Made(7, [40], 2, 128, 16, BF16)
    q = _randn(8, (2, 128 + 2), BF16)[:, :128].unsqueeze(0)
    odd = _randn(9, (2 * 128 + 1,), BF16)[1:].view(1, 2, 128)
    for x in (q, odd):
        got = pc.paged_attention(x, made.cache, made.table, made.lens)
        assert torch.equal(got, pc.paged_attention(x.clone(memory_format=torch.contiguous_format), made.cache, made.table,
                                                   made.lens))
    with pytest.raises(AttributeError):
        made.cache.k = made.cache.v


def test_rotary_of_more_tokens_than_one_grid_dimension_holds():
    """2^24 workgroups of 256 threads are 2^32 of them."""
    import paged_cache as pc
    T = (1 << 24) + 3
    q = torch.arange(T * 16, device=DEV, dtype=torch.int32).remainder_(509).to(BF16).view(T, 1, 16)
    positions, inv_freq = torch.arange(T, device=DEV, dtype=torch.int32), torch.ones(8, device=DEV)
    got, _ = pc.rotary(q, None, positions, inv_freq)
    for at in (0, (1 << 20) - 2, (1 << 23) + 5, T - 7):
        part, _ = pc.rotary(q[at:at + 7], None, positions[at:at + 7], inv_freq)
        assert torch.equal(got[at:at + 7], part)


def test_rotary_gradients_through_autograd():
    """Against the formula's gradient and against differences of the formula in 64 bits."""
    import paged_cache as pc
    q, k = _randn(8, (11, 4, 64), F32).requires_grad_(), _randn(9, (11, 2, 64), F32).requires_grad_()
    positions = torch.arange(22, device=DEV).reshape(2, 11) * 31
    inv_freq = (500.0 ** -(torch.arange(32) / 32.0)).to(DEV)
    wq, wk = _randn(10, (11, 4, 64), F32), _randn(11, (11, 2, 64), F32)
    a, b = pc.rotary(q, k, positions, inv_freq, (16, 16), 0.5, 1.25)
    ((a * wq).sum() + (b * wk).sum()).backward()
    _check_rotary(wq, q.grad, positions, inv_freq, (16, 16), 0.5, 1.25, True)
    _check_rotary(wk, k.grad, positions, inv_freq, (16, 16), 0.5, 1.25, True)
    x0 = q.detach().double().cpu()
    for t, h, d in ((0, 0, 0), (5, 3, 31), (10, 1, 63), (7, 2, 40)):
        step = torch.zeros_like(x0)
        step[t, h, d] = 1.0
        up, _ = ref.rotary(x0 + step, positions, inv_freq, (16, 16), 0.5, 1.25)
        down, _ = ref.rotary(x0 - step, positions, inv_freq, (16, 16), 0.5, 1.25)
        slope = float(((up - down) / 2 * wq.double().cpu()).sum())
        assert abs(float(q.grad[t, h, d]) - slope) <= 64 * U * (1 + abs(slope)) * 8
    # linear: the second derivative is that of the rotation again
    g, = torch.autograd.grad(pc.rotary(q, k, positions, inv_freq, (16, 16))[0], q, wq, create_graph=False)
    w = wq.clone().requires_grad_()
    g2, = torch.autograd.grad(pc.rotary(q, k, positions, inv_freq, (16, 16))[0], q, w, create_graph=True)
    assert torch.equal(g, g2)
    back, = torch.autograd.grad(g2, w, q.detach())
    _check_rotary(q, back, positions, inv_freq, (16, 16))


# ----------------------------------------------------------------------------------------- the cache
class Made:
    """A cache with random contents, pages shuffled, and tables of the given lengths (room: spare slots)."""

    def __init__(self, seed, lens, Hkv, D, ps, dtype, room=0, layout="head", spare=2, extra_width=0):
        g = torch.Generator().manual_seed(seed)
        need = [-(-(n + room) // ps) for n in lens]
        pages, width = sum(need) + spare, max(max(need), 1) + extra_width
        shape = (pages, Hkv, ps, D)
        if layout == "head":
            k, v = _randn(seed + 1, shape, dtype), _randn(seed + 2, shape, dtype)
        elif layout == "slot":                                # (pages, slots, heads, D) underneath
            k = _randn(seed + 1, (pages, ps, Hkv, D), dtype).transpose(1, 2)
            v = _randn(seed + 2, (pages, ps, Hkv, D), dtype).transpose(1, 2)
        else:                                                 # k and v of a page side by side
            kv = _randn(seed + 1, (pages, Hkv, 2, ps, D), dtype)
            k, v = kv[:, :, 0], kv[:, :, 1]
        weight = torch.rand((pages, Hkv, ps), generator=g).to(DEV)
        pos = torch.zeros((pages, Hkv, ps), dtype=torch.int32)
        ids = torch.randperm(pages, generator=g).tolist()
        self.rows, at = [], 0
        for n in need:
            self.rows.append(ids[at:at + n] + [-1] * (width - n))
            for c, p in enumerate(ids[at:at + n]):
                pos[p] = torch.arange(c * ps, (c + 1) * ps, dtype=torch.int32)
            at += n
        self.free = ids[at:]
        self.lens_host, self.ps = lens, ps
        self.table = torch.tensor(self.rows, dtype=torch.int32, device=DEV)
        self.lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
        import paged_cache as pc
        self.cache = pc.PagedCache(k, v, weight, pos.to(DEV))
        self.cap = width * ps

    def attend_ref(self, q, sm_scale, cap=None, lens=None):
        q4 = q if q.dim() == 4 else q[:, :, None]
        return ref.attend(q4, self.cache.k, self.cache.v, self.table.cpu(), lens or self.lens_host, sm_scale,
                          self.cap if cap is None else cap)


def _check_attend(made, q, got, want, lse=None, weight=None, weight0=None):
    out, want_lse, drawn, reach, score = want
    D = q.shape[-1]
    n = max(max(made.lens_host), 1)
    rel = 2 * (D + 8) * U * score + (n + 64) * U                                      # (B, H, Q)
    tiny = torch.finfo(q.dtype).smallest_normal
    tol = (rel[..., None] * reach + _half_step(q.dtype) * out.abs()) * 1.01 + tiny * _half_step(q.dtype)
    err = (got.double().cpu().reshape(out.shape) - out).abs()
    assert torch.all(err <= tol), f"out off by {err.max().item():.3e}, {(err / tol.clamp(min=1e-300)).max().item():.2f} of the bound"
    if lse is not None:
        lse = lse.double().cpu().reshape(want_lse.shape)
        fine = torch.isfinite(want_lse)
        assert torch.equal(torch.isfinite(lse), fine) and torch.all(lse[~fine] == float("-inf"))
        assert torch.all((lse - want_lse).abs()[fine] <= (rel + 4 * U * (1 + want_lse.abs()))[fine])
    if weight is not None:
        rows = q.shape[1] * (q.shape[2] if q.dim() == 4 else 1) // made.cache.kv_heads
        grow = weight0.double().cpu()
        touched = torch.zeros_like(grow, dtype=torch.bool)
        for (b, h), w in drawn.items():
            for j0 in range(0, len(w), made.ps):
                p = int(made.table[b, j0 // made.ps])
                if 0 <= p < grow.shape[0]:
                    m = min(made.ps, len(w) - j0)
                    grow[p, h, :m] += w[j0:j0 + m]
                    touched[p, h, :m] = True
        err = (weight.double().cpu() - grow).abs()
        tol = (2 * rel.max() + (rows + 4) * U) * grow * 1.01
        assert torch.all(err[touched] <= tol[touched]), f"weight off by {err.max().item():.3e}"
        assert torch.equal(weight.cpu()[~touched], weight0.cpu()[~touched]), "a weight outside the sequences changed"


ATTEND = [
    # lens, H, Hkv, Q, D, page size, dtype, layout
    ([1], 8, 2, 1, 128, 16, BF16, "head"),
    ([0, 1, 2, 15, 16, 17], 4, 2, 1, 64, 16, F16, "slot"),
    ([31, 32, 33, 63, 64, 65, 127, 128, 129], 8, 8, 1, 128, 32, BF16, "pair"),
    ([1000, 0, 257, 511], 32, 8, 1, 128, 16, BF16, "head"),
    ([300, 77], 6, 2, 1, 128, 1, F32, "head"),
    ([700, 1, 333], 7, 7, 1, 64, 64, F32, "slot"),
    ([2500], 16, 1, 1, 128, 256, F16, "head"),
    ([513, 90], 71, 1, 1, 64, 8, BF16, "head"),
    ([40, 3, 0, 129], 8, 2, 5, 128, 16, BF16, "head"),
    ([200, 31], 6, 3, 16, 64, 2, F32, "pair"),
    ([600, 33, 5], 28, 4, 32, 128, 32, F16, "slot"),
    ([170], 24, 1, 33, 128, 128, BF16, "head"),
    ([5000, 4097], 8, 2, 1, 128, 64, BF16, "head"),
    ([1500, 7], 4, 2, 40, 128, 16, F32, "head"),              # 80 rows a kv head, fp32
    ([3, 900], 40, 1, 1, 128, 16, F16, "slot"),               # three row tiles, one query
    ([1024, 1023], 4, 4, 1, 64, 16, F32, "head"),
] + [([100 + 13 * i] * 3 + [0] * (i % 2), 4, 2, 1 + i % 2, 64, 16, BF16, "head") for i in range(2)] + [
    ([1 + (37 * i) % 90 for i in range(150)], 4, 2, 1, 64, 16, BF16, "head"),      # more sequences than lanes
    ([1 + (37 * i) % 90 for i in range(150)] + [1200], 4, 2, 1, 64, 16, BF16, "head"),
    ([700, 9, 0, 1301], 8, 2, 16, 128, 16, BF16, "head"),      # 64 rows a kv head
    ([333, 40], 16, 4, 16, 64, 8, F16, "pair"),
    ([610, 90], 8, 2, 20, 128, 4, BF16, "slot"),               # 80 rows, pages of less than 8
]


@pytest.mark.parametrize("case", range(len(ATTEND)))
@pytest.mark.parametrize("accumulate", [False, True])
def test_attention_against_the_definition(case, accumulate):
    import paged_cache as pc
    lens, H, Hkv, Q, D, ps, dtype, layout = ATTEND[case]
    print(f"[case] attend {ATTEND[case]} accumulate={accumulate}", flush=True)
    made = Made(10 * case, lens, Hkv, D, ps, dtype, layout=layout, extra_width=case % 3)
    q = _randn(10 * case + 5, (len(lens), H, Q, D) if Q > 1 or case % 2 else (len(lens), H, D), dtype, 1.5)
    weight0 = made.cache.weight.clone()
    kw = {"accumulate": accumulate, "want_lse": case % 2 == 0}
    if case % 3 == 1:
        kw["max_len"] = max(max(lens), 1)
    got = pc.paged_attention(q, made.cache, made.table, made.lens, **kw)
    got, lse = got if kw["want_lse"] else (got, None)
    assert got.shape == q.shape and got.dtype == q.dtype
    want = made.attend_ref(q, 1.0 / math.sqrt(D))
    _check_attend(made, q, got, want, lse, made.cache.weight if accumulate else None, weight0)
    if not accumulate:
        assert torch.equal(made.cache.weight, weight0)


@pytest.mark.parametrize("Q", [1, 3])
def test_weights_of_any_alignment(Q):
    import paged_cache as pc
    made = Made(90, [1500, 3, 2049], 2, 64, 16, BF16)
    c = made.cache
    flat = torch.zeros(c.weight.numel() + 1, device=DEV)
    shifted = flat[1:].view(c.weight.shape)
    shifted.copy_(c.weight)
    made.cache = pc.PagedCache(c.k, c.v, shifted, c.pos)
    q = _randn(91, (3, 8, Q, 64), BF16)
    before = shifted.clone()
    got, lse = pc.paged_attention(q, made.cache, made.table, made.lens, accumulate=True, want_lse=True)
    _check_attend(made, q, got, made.attend_ref(q, 0.125), lse, shifted, before)
    aligned = pc.PagedCache(c.k, c.v, before.clone(), c.pos)
    pc.paged_attention(q, aligned, made.table, made.lens, accumulate=True)
    assert torch.equal(aligned.weight, shifted)


def test_attention_of_strided_queries_scales_and_a_short_bound():
    import paged_cache as pc
    made = Made(200, [300, 90], 2, 64, 16, BF16)
    wide = _randn(201, (2, 3, 8, 64), BF16)                   # tokens before heads, as a projection leaves them
    q = wide.transpose(1, 2)
    for scale in (0.0, -0.3, 2.0):
        got, lse = pc.paged_attention(q, made.cache, made.table, made.lens, sm_scale=scale, want_lse=True)
        _check_attend(made, q, got, made.attend_ref(q, scale), lse)
    got = pc.paged_attention(q, made.cache, made.table, made.lens, max_len=100)      # a length past the bound
    _check_attend(made, q, got, made.attend_ref(q, 0.125, cap=100))
    long = torch.tensor([10 ** 6, -5], dtype=torch.int32, device=DEV)                # past the table, below 0
    got = pc.paged_attention(q, made.cache, made.table, long)
    _check_attend(made, q, got, made.attend_ref(q, 0.125, lens=[10 ** 6, -5]))
    got = pc.paged_attention(q, made.cache, made.table.long(), made.lens.long())     # 64-bit tables are converted
    _check_attend(made, q, got, made.attend_ref(q, 0.125))
    odd = _randn(202, (2, 8, 67), BF16)[..., 1:65]            # rows that are not 16-byte aligned
    _check_attend(made, odd, pc.paged_attention(odd, made.cache, made.table, made.lens), made.attend_ref(odd, 0.125))


@pytest.mark.parametrize("Q,dtype", [(1, BF16), (4, BF16), (3, F32), (1, F16), (40, BF16), (20, F16), (40, F32)])
def test_attention_ignores_what_it_does_not_see(Q, dtype):
    """NaN and infinities behind the sequences, in pages of no table, and in keys that the earlier
    queries of a call do not see; entries that are no page."""
    import paged_cache as pc
    made = Made(300, [130, 70, 33, 64], 2, 64, 32, dtype, extra_width=1)
    q = _randn(301, (4, 8, Q, 64), dtype)
    table = made.table.clone()
    table[0, 1], table[2, 0], table[2, 1] = -1, 10 ** 6, -7   # sequence 2 has no page at all
    made.table = table
    want = made.attend_ref(q, 0.125)
    clean = pc.paged_attention(q, made.cache, table, made.lens)
    _check_attend(made, q, clean, want)
    assert torch.all(clean[2] == 0)
    bad = [float("nan"), float("inf"), float("-inf")]
    for p in made.free:
        made.cache.k[p], made.cache.v[p] = bad[0], bad[1]
    for i, n in enumerate(made.lens_host):
        if n % 32 and int(table[i, n // 32]) >= 0 and int(table[i, n // 32]) < made.cache.pages:
            made.cache.k[int(table[i, n // 32]), :, n % 32:] = bad[i % 3]
            made.cache.v[int(table[i, n // 32]), :, n % 32:] = bad[(i + 1) % 3]
    weight0 = made.cache.weight.clone()
    again, lse = pc.paged_attention(q, made.cache, table, made.lens, accumulate=True, want_lse=True)
    assert torch.equal(again, clean)
    _check_attend(made, q, again, want, lse, made.cache.weight, weight0)
    # the newest key of sequence 1 is NaN: only its own query sees it
    p = int(table[1, 69 // 32])
    made.cache.v[p, :, 69 % 32] = bad[0]
    again = pc.paged_attention(q, made.cache, table, made.lens)
    assert torch.equal(again[:, :, :Q - 1], clean[:, :, :Q - 1]) and torch.isnan(again[1, :, Q - 1]).all()
    assert torch.equal(again[[0, 2, 3], :, Q - 1], clean[[0, 2, 3], :, Q - 1])
    made.cache.v[p, :, 69 % 32] = 0.0
    made.cache.k[p, :, 69 % 32] = bad[0]
    again = pc.paged_attention(q, made.cache, table, made.lens)
    assert torch.equal(again[:, :, :Q - 1], clean[:, :, :Q - 1]) and torch.isnan(again[1, :, Q - 1]).all()


def test_attention_of_extreme_scores():
    import paged_cache as pc
    made = Made(310, [100, 40, 300], 1, 64, 16, F32)
    q = torch.zeros(3, 2, 64, device=DEV)
    q[:, :, 0] = 1.0
    k = made.cache.k
    k.zero_()
    rows = [made.rows[b] for b in range(3)]
    k[rows[0][2], 0, 3, 0] = 3.0e38                           # one key takes all
    k[rows[1][:3], 0, :, 0] = float("-inf")                   # a row whose every score is -inf: zeros
    k[rows[2][:19], 0, :, 0] = -3.0e38                        # equal scores far below zero
    got, lse = pc.paged_attention(q, made.cache, made.table, made.lens, sm_scale=1.0, want_lse=True)
    v = made.cache.v
    assert torch.equal(got[0, 0], v[rows[0][2], 0, 3]) and torch.equal(got[0, 1], got[0, 0])
    assert torch.all(got[1] == 0) and torch.all(lse[1] == float("-inf"))
    mean = ref.keys_of(v, rows[2], 300, 16, 0)[0].mean(0)
    assert torch.all((got[2].double().cpu() - mean).abs() <= 364 * U * 4)
    k[rows[0][2], 0, 3, 0] = float("inf")                     # inf - inf: NaN, as the softmax says
    got = pc.paged_attention(q, made.cache, made.table, made.lens, sm_scale=1.0)
    assert torch.isnan(got[0]).all() and torch.isfinite(got[1:]).all()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("Q", [1, 3])
def test_attention_of_infinite_values(dtype, Q):
    """A value of infinity makes its dim infinite for every query that sees its key, with either sign NaN, and
    leaves the other dims alone."""
    import paged_cache as pc
    inf = float("inf")
    for lens in ([600, 50], [3000, 50]):                      # one launch, and split
        made = Made(350, lens, 2, 64, 16, dtype)
        q = _randn(351, (2, 8, Q, 64), dtype)
        clean = pc.paged_attention(q, made.cache, made.table, made.lens)
        p, v = made.rows[0][2], made.cache.v
        v[p, 0, 5, 7], v[p, 0, 6, 9], v[p, 0, 7, 9], v[p, 0, 8, 11] = inf, inf, -inf, -inf
        v[made.rows[1][0], 1, 0, 0] = inf
        got = pc.paged_attention(q, made.cache, made.table, made.lens).float()
        assert torch.all(got[0, :4, :, 7] == inf) and torch.isnan(got[0, :4, :, 9]).all()
        assert torch.all(got[0, :4, :, 11] == -inf) and torch.all(got[1, 4:, :, 0] == inf)
        want = clean.float()
        for x in (got, want):
            x[0, :4, :, [7, 9, 11]] = 0.0
            x[1, 4:, :, 0] = 0.0
        # P whole or in two parts: both within the bound of the definition, so within twice that of each other
        made.cache.v.nan_to_num_(0.0, 0.0, 0.0)
        out, _, _, reach, score = made.attend_ref(q, 0.125)
        rel = 2 * 72 * U * score + (max(lens) + 64) * U
        tol = 2 * (rel[..., None] * reach + _half_step(dtype) * out.abs()) * 1.01 + torch.finfo(dtype).smallest_normal
        assert torch.all((got - want).abs().cpu().double() <= tol)


def test_attention_past_4_gib_of_cache():
    """Pages whose rows lie beyond 32-bit byte offsets."""
    import paged_cache as pc
    ps, D, Hkv = 128, 128, 8
    pages = 20000                                             # 5.2 GB of keys, as many of values
    k = torch.empty((pages, Hkv, ps, D), dtype=BF16, device=DEV)
    v = torch.empty_like(k)
    use = [19999, 3, 18001, 17777]
    for i, p in enumerate(use):
        k[p], v[p] = _randn(320 + i, (Hkv, ps, D), BF16), _randn(330 + i, (Hkv, ps, D), BF16)
    made = Made(340, [3 * ps + 17], Hkv, D, ps, BF16)
    made.cache = pc.PagedCache(k, v, torch.zeros((pages, Hkv, ps), device=DEV),
                               torch.arange(ps, dtype=torch.int32, device=DEV).expand(pages, Hkv, ps).contiguous())
    made.table = torch.tensor([use], dtype=torch.int32, device=DEV)
    made.cap = 4 * ps
    q = _randn(341, (1, 16, D), BF16)
    got = pc.paged_attention(q, made.cache, made.table, made.lens, accumulate=True)
    _check_attend(made, q, got, made.attend_ref(q, 1 / math.sqrt(D)))
    new = _randn(342, (1, Hkv, D), BF16)
    lens = pc.cache_append(made.cache, new, new, made.table, made.lens)
    assert int(lens) == 3 * ps + 18 and torch.equal(k[17777, :, 17], new[0])
    before = k[19999, :, 5].clone()
    pc.cache_evict(made.cache, made.table, lens, 2 * ps, 16, 16, dst_table=torch.tensor([[19000, 18999]], device=DEV))
    assert torch.equal(k[19000, :, 5], before)                # a forced key: positions below 16


# -------------------------------------------------------------------------------------------- append
@pytest.mark.parametrize("ps,D,dtype,layout", [(16, 128, BF16, "head"), (1, 64, F32, "slot"), (64, 64, F16, "pair")])
def test_append_against_the_definition(ps, D, dtype, layout):
    import paged_cache as pc
    lens, new = [0, 5, 63, 64, 1], [3, 0, 70, 1, 20]
    made = Made(400, lens, 3, D, ps, dtype, room=70, layout=layout)
    starts = [2]
    for n in new:
        starts.append(starts[-1] + n)
    T = starts[-1] + 4                                        # rows of no sequence in front and behind
    k, v = _randn(401, (T, 3, D), dtype), _randn(402, (3, T, D), dtype).transpose(0, 1)
    seen = torch.tensor([0, 500, 63, 64, 9], dtype=torch.int32, device=DEV)
    want = [x.cpu().clone() for x in (made.cache.k, made.cache.v, made.cache.weight, made.cache.pos)]
    for b, n in enumerate(new):
        for i in range(n):
            p, s = made.rows[b][(lens[b] + i) // ps], (lens[b] + i) % ps
            want[0][p, :, s], want[1][p, :, s] = k[starts[b] + i].cpu(), v[starts[b] + i].cpu()
            want[2][p, :, s], want[3][p, :, s] = 0.0, int(seen[b]) + i
    got = pc.cache_append(made.cache, k, v, made.table, made.lens, torch.tensor(starts, device=DEV), seen)
    assert got.tolist() == [a + b for a, b in zip(lens, new)] and made.lens.tolist() == lens
    for x, w in zip((made.cache.k, made.cache.v, made.cache.weight, made.cache.pos), want):
        assert torch.equal(x.cpu(), w)


def test_append_stops_at_the_table_and_at_missing_pages():
    import paged_cache as pc
    made = Made(410, [16, 30, 8], 2, 64, 16, F32, extra_width=0)      # tables 2 wide; sequences 0 and 2 own one page
    before = [x.clone() for x in (made.cache.k, made.cache.v, made.cache.weight, made.cache.pos)]
    k = _randn(411, (9, 2, 64), F32)
    starts = torch.tensor([0, 3, 8, 9], dtype=torch.int32, device=DEV)
    got = pc.cache_append(made.cache, k, k, made.table, made.lens, starts)
    assert got.tolist() == [19, 32, 9]                        # 30 + 5 stops at 32 slots
    p = made.rows[1][1]
    before[0][p, :, 14:16] = before[1][p, :, 14:16] = k[3:5].transpose(0, 1)
    before[2][p, :, 14:16], before[3][p, :, 14:16] = 0.0, torch.tensor([30, 31], dtype=torch.int32, device=DEV)
    p = made.rows[2][0]
    before[0][p, :, 8] = before[1][p, :, 8] = k[8]
    before[2][p, :, 8], before[3][p, :, 8] = 0.0, 8
    for x, w in zip((made.cache.k, made.cache.v, made.cache.weight, made.cache.pos), before):
        assert torch.equal(x, w)
    got = pc.cache_append(pc.PagedCache(made.cache.k, made.cache.v), k[:0], k[:0], made.table, made.lens,
                          torch.zeros(4, dtype=torch.int32, device=DEV))
    assert got.tolist() == [16, 30, 8]


# ------------------------------------------------------------------------------------------ eviction
EVICT = [
    # lens, Hkv, D, page size, dtype, budget, n_global, n_local, layout
    ([100, 7, 64, 65, 0], 2, 64, 16, BF16, 64, 4, 8, "head"),
    ([1000], 3, 128, 32, F16, 999, 4, 32, "slot"),
    ([3000, 1500, 40], 2, 64, 8, F32, 500, 0, 0, "head"),
    ([2049, 1025], 1, 128, 1, BF16, 1, 0, 1, "head"),
    ([300, 290], 2, 64, 128, BF16, 200, 150, 150, "pair"),    # more forced keys than the budget holds
    ([5000], 1, 64, 64, F32, 4096, 16, 16, "head"),
    ([30011, 12], 1, 64, 16, BF16, 700, 4, 32, "head"),       # words beyond LDS
    ([20000], 2, 64, 128, BF16, 19990, 0, 5, "head"),         # few moves, found in a long sequence
]


@pytest.mark.parametrize("case", range(len(EVICT)))
@pytest.mark.parametrize("move", [False, True])
def test_eviction_against_the_definition(case, move):
    import paged_cache as pc
    lens, Hkv, D, ps, dtype, budget, n_global, n_local, layout = EVICT[case]
    print(f"[case] evict {EVICT[case]} dst_table={move}", flush=True)
    left = [min(n, budget) for n in lens]
    spare = sum(-(-m // ps) for m in left) + 1
    made = Made(500 + 10 * case, lens, Hkv, D, ps, dtype, layout=layout, spare=spare)
    w = made.cache.weight
    w.copy_((w * 50).round() / 50 if case % 2 == 0 else w)    # many equal weights
    if case == 2:
        for x, at in ((float("nan"), 40), (float("inf"), 50), (-1.0, 60), (-0.0, 70), (0.0, 71), (float("-inf"), 72)):
            w[made.rows[0][at], 1, :4] = x
    perm = torch.randperm(made.ps, generator=torch.Generator().manual_seed(1)).to(DEV)
    made.cache.pos.copy_(made.cache.pos[:, :, perm])          # slots out of order, as after an eviction
    dst, free = None, iter(made.free)
    if move:
        width = max(1, -(-min(budget, max(lens)) // ps))
        dst = [[next(free) for _ in range(-(-m // ps))] for m in left]
        dst = torch.tensor([r + [-1] * (width - len(r)) for r in dst], dtype=torch.int32, device=DEV)
    want = ref.evict(made.cache.k, made.cache.v, w, made.cache.pos, made.table, lens, budget, n_global, n_local,
                     made.cap, dst)
    kw = {"max_len": max(lens)} if case % 2 else {}
    got = pc.cache_evict(made.cache, made.table, made.lens, budget, n_global, n_local, dst, **kw)
    assert got.tolist() == left and made.lens.tolist() == lens
    for name, x, y in zip(("k", "v", "weight", "pos"), (made.cache.k, made.cache.v, w, made.cache.pos), want):
        assert torch.equal(x.cpu().view(torch.uint8), y.view(torch.uint8)), name


def test_eviction_of_numbers_beyond_32_bits():
    """A budget or window that no length reaches keeps everything, and one below zero is refused."""
    import paged_cache as pc
    made = Made(700, [90, 20], 2, 64, 16, BF16)
    before = made.cache.k.clone(), made.cache.weight.clone()
    for kw in ({"budget": 2 ** 32 + 5}, {"budget": 2 ** 31}, {"budget": 95, "n_local": 2 ** 32 + 1, "max_len": 2 ** 33}):
        assert pc.cache_evict(made.cache, made.table, made.lens, **kw).tolist() == [90, 20]
    assert torch.equal(made.cache.k, before[0]) and torch.equal(made.cache.weight, before[1])
    for kw in ({"budget": -2 ** 32 + 5}, {"budget": 5, "n_global": -2 ** 32 + 5}, {"budget": 5, "max_len": -2 ** 32 + 5}):
        with pytest.raises(RuntimeError):
            pc.cache_evict(made.cache, made.table, made.lens, **kw)


def test_eviction_with_weights_and_positions_of_any_alignment():
    import paged_cache as pc
    made = Made(580, [300, 64], 3, 64, 16, BF16)
    c = made.cache
    wide_w = torch.zeros((c.pages, 4, 19), device=DEV)
    wide_p = torch.zeros((c.pages, 5, 17), dtype=torch.int32, device=DEV)
    w, p = wide_w[:, 1:, 3:], wide_p[:, :3, 1:]               # strides and bases off 16 bytes
    w.copy_(c.weight)
    p.copy_(c.pos)
    want = ref.evict(c.k, c.v, w, p, made.table, [300, 64], 100, 4, 8, made.cap)
    other = pc.PagedCache(c.k, c.v, w, p)
    pc.cache_evict(other, made.table, made.lens, 100, 4, 8)
    for x, y in zip((c.k, c.v, w, p), want):
        assert torch.equal(x.cpu(), y)
    assert torch.all(wide_w[:, 0] == 0) and torch.all(wide_w[:, :, :3] == 0) and torch.all(wide_p[:, 3:] == 0)


def test_a_long_eviction_in_a_graph():
    import paged_cache as pc
    made, other = Made(585, [20000, 900], 2, 64, 16, BF16), Made(585, [20000, 900], 2, 64, 16, BF16)
    left = pc.cache_evict(made.cache, made.table, made.lens, 600, 4, 8)
    fields = lambda m: (m.cache.k, m.cache.v, m.cache.weight, m.cache.pos)           # noqa: E731
    start = [x.clone() for x in fields(other)]
    pc.cache_evict(other.cache, other.table, other.lens, 600, 4, 8)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = pc.cache_evict(other.cache, other.table, other.lens, 600, 4, 8)
    for _ in range(3):
        for x, y in zip(fields(other), start):
            x.copy_(y)
        got.zero_()
        pc.cache_evict(made.cache, made.table, left, 600, 4, 8)                      # eager work in between: no moves
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, left)
        for x, y in zip(fields(other), fields(made)):
            assert torch.equal(x, y)


def test_eviction_of_missing_pages():
    """Keys without a page go first; nothing is written outside the sequence's pages."""
    import paged_cache as pc
    made = Made(590, [100, 90], 2, 64, 16, F32)
    table = made.table.clone()
    table[0, 1], table[1, 5] = -1, 9999
    args = (made.cache.k, made.cache.v, made.cache.weight, made.cache.pos, table, [100, 90], 70, 4, 4, made.cap)
    want = ref.evict(*args)
    pc.cache_evict(made.cache, table, made.lens, 70, 4, 4)
    for x, y in zip((made.cache.k, made.cache.v, made.cache.weight, made.cache.pos), want):
        assert torch.equal(x.cpu(), y)


# ------------------------------------------------------------------------------------------- together
def _step(pc, made, q, k, v, lens, seen, inv_freq, budget):
    q, k = pc.rotary(q, k, seen, inv_freq)
    lens = pc.cache_append(made.cache, k, v, made.table, lens, seen=seen)
    out = pc.paged_attention(q, made.cache, made.table, lens, accumulate=True)
    return out, pc.cache_evict(made.cache, made.table, lens, budget, 2, 4)


def test_decoding_at_a_budget_matches_the_definitions_step_by_step():
    """A batch decodes until its caches are full and then evicts a key a step: after each step the state is
    what the definitions make of the state before it."""
    import paged_cache as pc
    H, Hkv, D, ps, budget = 8, 2, 64, 8, 24
    made = Made(600, [20, 24, 0], Hkv, D, ps, F32, room=0, spare=12, extra_width=1)
    rows, free = [r[:] for r in made.rows], iter(made.free)
    for r in rows:
        r[:] = [p if p >= 0 else next(free) for p in r][:4]
    made.rows, made.table = rows, torch.tensor(rows, dtype=torch.int32, device=DEV)
    made.cap = made.table.shape[1] * ps
    for c in range(made.table.shape[1]):
        made.cache.pos[made.table[:, c].long()] = torch.arange(c * ps, (c + 1) * ps, dtype=torch.int32, device=DEV)
    inv_freq = (10000.0 ** -(torch.arange(32) / 32.0)).to(DEV)
    lens, seen = made.lens, made.lens.clone()
    for t in range(7):
        q, k, v = (_randn(610 + 3 * t + i, (3, n, D), F32) for i, n in enumerate((H, Hkv, Hkv)))
        qr, kr = pc.rotary(q, k, seen, inv_freq)
        host = [x.cpu().clone() for x in (made.cache.k, made.cache.v, made.cache.weight, made.cache.pos)]
        n0 = lens.tolist()
        for b, n in enumerate(n0):
            p, s = rows[b][n // ps], n % ps
            host[0][p, :, s], host[1][p, :, s], host[2][p, :, s] = kr[b].cpu(), v[b].cpu(), 0.0
            host[3][p, :, s] = int(seen[b])
        out, lens = _step(pc, made, q, k, v, lens, seen, inv_freq, budget)
        grown = [n + 1 for n in n0]
        want = ref.attend(qr[:, :, None].cpu(), host[0], host[1], made.table.cpu(), grown, 0.125, made.cap)
        made.lens_host = grown
        _check_attend(made, q, out, want)
        for (b, h), w in want[2].items():
            for j in range(len(w)):
                host[2][rows[b][j // ps], h, j % ps] += float(w[j])
        k2, v2, w2, p2, left = ref.evict(*host, made.table.cpu(), grown, budget, 2, 4, made.cap)
        assert lens.tolist() == left.tolist()
        assert torch.equal(made.cache.pos.cpu(), p2) and torch.equal(made.cache.k.cpu(), k2)
        assert torch.equal(made.cache.v.cpu(), v2)
        # 2 (D + 8) u S + (n + 64) u with S < 11 for these inputs
        assert float(want[4].max()) < 11 and torch.all((made.cache.weight.cpu() - w2).abs() <= 1e-4 * w2.abs() + 1e-9)
        seen = seen + 1


def test_step_in_a_graph_replays_as_eager_steps():
    """The whole step captured: replays, with eager work between them, end in the same state, bit for bit, as
    eager steps on a copy."""
    import paged_cache as pc
    H, Hkv, D, ps, budget = 16, 4, 128, 16, 160
    print("[case] the step in a graph", flush=True)

    def make():
        made = Made(700, [160, 200, 75], Hkv, D, ps, BF16, room=ps)
        return made, made.lens.clone(), torch.tensor([900, 901, 75], dtype=torch.int32, device=DEV)
    inv_freq = (10000.0 ** -(torch.arange(64) / 64.0)).to(DEV)
    inputs = [[_randn(710 + 3 * t + i, (3, n, D), BF16) for i, n in enumerate((H, Hkv, Hkv))] for t in range(5)]
    made, lens, seen = make()
    outs = []
    for q, k, v in inputs:
        out, lens = _step(pc, made, q, k, v, lens, seen, inv_freq, budget)
        seen = seen + 1
        outs.append(out)
    other, glens, gseen = make()
    bufs = [x.clone() for x in inputs[0]]
    g = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g):
        gout, new = _step(pc, other, *bufs, glens, gseen, inv_freq, budget)
        glens.copy_(new)
        gseen.add_(1)
    for t, x in enumerate(inputs):
        for a, b in zip(bufs, x):
            a.copy_(b)
        pc.paged_attention(inputs[0][0], made.cache, made.table, lens)           # eager work in between
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(gout, outs[t]), f"replay {t}"
    assert torch.equal(glens, lens) and torch.equal(gseen, seen)
    for a, b in ((other.cache.k, made.cache.k), (other.cache.v, made.cache.v), (other.cache.weight, made.cache.weight),
                 (other.cache.pos, made.cache.pos)):
        assert torch.equal(a, b)


def test_two_streams_at_once():
    import paged_cache as pc
    a, b = Made(800, [3000, 100], 4, 128, 16, BF16), Made(820, [700, 2900], 2, 64, 32, F16)
    qa, qb = _randn(801, (2, 16, 128), BF16), _randn(821, (2, 16, 2, 64), F16)
    ra = pc.paged_attention(qa, a.cache, a.table, a.lens)
    rb = pc.paged_attention(qb, b.cache, b.table, b.lens)
    torch.cuda.synchronize()
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(4):
        with torch.cuda.stream(s):
            x = pc.paged_attention(qa, a.cache, a.table, a.lens, accumulate=True)
        with torch.cuda.stream(t):
            y = pc.paged_attention(qb, b.cache, b.table, b.lens, accumulate=True)
        torch.cuda.synchronize()
        assert torch.equal(x, ra) and torch.equal(y, rb)


def test_shared_pages_are_read_by_many_sequences():
    import paged_cache as pc
    made = Made(850, [200], 2, 64, 16, BF16)
    q = _randn(851, (5, 4, 64), BF16)
    made.table = made.table.expand(5, -1)                     # stride 0: one table row for all
    made.lens_host = [200, 13, 100, 0, 199]
    made.lens = torch.tensor(made.lens_host, dtype=torch.int32, device=DEV)
    got = pc.paged_attention(q, made.cache, made.table, made.lens)
    _check_attend(made, q, got, made.attend_ref(q, 0.125))


# ------------------------------------------------------------------------------------------ refusals
def test_refusals_on_the_device():
    import paged_cache as pc
    made = Made(900, [20, 20], 2, 64, 16, BF16)
    c, t, n = made.cache, made.table, made.lens
    q = _randn(901, (2, 4, 64), BF16)
    k = _randn(902, (2, 2, 64), BF16)
    with pytest.raises(TypeError):
        pc.paged_attention(q.float(), c, t, n)
    with pytest.raises(ValueError):
        pc.paged_attention(q[:1], c, t, n)
    with pytest.raises(ValueError):
        pc.paged_attention(q[..., :32], c, t, n)
    with pytest.raises(RuntimeError, match="multiple"):
        pc.paged_attention(_randn(1, (2, 3, 64), BF16), c, t, n)
    with pytest.raises(RuntimeError, match="HIP device"):
        pc.paged_attention(q.cpu(), c, t, n)
    with pytest.raises(RuntimeError, match="weight"):
        pc.paged_attention(q, pc.PagedCache(c.k, c.v), t, n, accumulate=True)
    with pytest.raises(RuntimeError, match="weight"):
        pc.cache_evict(pc.PagedCache(c.k, c.v), t, n, 8)
    with pytest.raises(RuntimeError, match="budget"):
        pc.cache_evict(c, t, n, 0)
    with pytest.raises(RuntimeError, match="dst_table"):
        pc.cache_evict(c, t, n, 20, dst_table=t[:, :1])
    with pytest.raises(ValueError):
        pc.cache_append(c, k[:, :1], k[:, :1], t, n)
    with pytest.raises(RuntimeError, match="starts"):
        pc.cache_append(c, k[:1], k[:1], t, n)
    with pytest.raises(ValueError):
        pc.cache_append(c, k, k, t, n, starts=n)
    with pytest.raises(ValueError):
        pc.cache_append(c, k, k, t, n[:1])
    with pytest.raises(TypeError):
        pc.PagedCache(c.k, c.v, c.weight.double())
    with pytest.raises(ValueError):
        pc.PagedCache(c.k, c.v[:1])
    with pytest.raises(RuntimeError, match="page_size"):
        odd = torch.zeros(3, 2, 12, 64, dtype=BF16, device=DEV)
        pc.paged_attention(q, pc.PagedCache(odd, odd), t, n)
    with pytest.raises(RuntimeError, match="head_dim"):
        odd = torch.zeros(3, 2, 16, 96, dtype=BF16, device=DEV)
        pc.paged_attention(_randn(1, (2, 4, 96), BF16), pc.PagedCache(odd, odd), t, n)
    inv = torch.ones(32, device=DEV)
    with pytest.raises(ValueError):
        pc.rotary(q, k, torch.zeros((2, 2), dtype=torch.int32, device=DEV), inv)
    with pytest.raises(ValueError):
        pc.rotary(q, k, torch.zeros((2, 2), dtype=torch.int32, device=DEV), inv, (16, 8))
    with pytest.raises(TypeError):
        pc.rotary(q, k, torch.zeros(2, dtype=torch.float64, device=DEV), inv)
    with pytest.raises(RuntimeError, match="sections"):
        pc.rotary(q, k, torch.zeros(2, dtype=torch.int32, device=DEV), torch.ones(12, device=DEV))
