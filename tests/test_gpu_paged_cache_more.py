"""GPU: the paged cache's operators where their work is divided among many workgroups, at numbers beyond 32 bits, at
large scores and values, and under forward-mode differentiation.

Tolerances as in test_gpu_paged_cache.py (u = 2^-24): with S the sum of a row's |q_d k_jd| times sm_scale, its largest
over the keys, a probability carries a factor within rel = 2 (D + 8) u S + (n + 64) u of 1.
"""
import math

import pytest
import torch
import torch.autograd.forward_ad as fwad

import paged_ref as ref
from test_gpu_paged_cache import BF16, DEV, F16, F32, U, Made, _check_rotary, _half_step, _randn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _need_gpu():
    if not torch.cuda.is_available():
        pytest.skip("no HIP device")
    import _sta_native
    _sta_native.lib()


# -------------------------------------------------------------------------------------------- rotary
def test_rotary_forward_mode_on_the_device():
    import paged_cache as pc
    q, k, tq = _randn(1, (9, 4, 64), F32), _randn(2, (9, 2, 64), F32), _randn(3, (9, 4, 64), F32)
    positions = torch.arange(18, device=DEV).reshape(2, 9) * 31
    inv_freq = (500.0 ** -(torch.arange(32) / 32.0)).to(DEV)
    plain = pc.rotary(q, k, positions, inv_freq, (16, 16), 0.5, 1.25)
    with fwad.dual_level():
        a, b = pc.rotary(fwad.make_dual(q, tq), k, positions, inv_freq, (16, 16), 0.5, 1.25)
        a, b = fwad.unpack_dual(a), fwad.unpack_dual(b)
    assert torch.equal(a.primal, plain[0]) and torch.equal(b.primal, plain[1])
    _check_rotary(tq, a.tangent, positions, inv_freq, (16, 16), 0.5, 1.25)
    assert b.tangent is None or torch.all(b.tangent == 0)


# ------------------------------------------------------------------------------- numbers beyond 32 bits
def test_lengths_and_pages_of_64_bits():
    """Lengths beyond 32 bits count as the table's end, pages beyond them as none, tokens seen stay the largest number."""
    import paged_cache as pc
    made = Made(900, [90, 40], 2, 64, 16, BF16)
    q = _randn(901, (2, 4, 64), BF16)
    far = torch.tensor([2 ** 32 + 5, -2 ** 32 + 5], device=DEV)
    table = made.table.long()
    holes = table.clone()
    holes[0, 1], holes[0, 2] = holes[0, 1] + 2 ** 32, holes[0, 2] - 2 ** 32
    want = pc.paged_attention(q, made.cache, made.table, torch.tensor([made.cap, 0], dtype=torch.int32, device=DEV))
    assert torch.equal(pc.paged_attention(q, made.cache, table, far), want)
    gone = made.table.clone()
    gone[0, 1:3] = -1
    want = pc.paged_attention(q, made.cache, gone, made.lens)
    assert torch.equal(pc.paged_attention(q, made.cache, holes, made.lens.long()), want)
    assert pc.cache_evict(made.cache, table, far, 2 ** 20).tolist() == [made.cap, 0]
    k = _randn(902, (2, 2, 64), BF16)
    before = made.cache.k.clone()
    assert pc.cache_append(made.cache, k, k, table, far).tolist() == [made.cap, 1]
    p = made.rows[1][0]
    assert torch.equal(made.cache.k[p, :, 0], k[1])
    before[p, :, 0] = k[1]
    assert torch.equal(made.cache.k, before)


def test_tokens_seen_stop_at_the_largest_number():
    """pos is seen + i as far as 32 bits go; it does not wrap into the first tokens, which eviction always keeps."""
    import paged_cache as pc
    made = Made(910, [0, 0], 1, 64, 16, BF16, room=16)
    k = _randn(911, (8, 1, 64), BF16)
    starts = torch.tensor([0, 4, 8], dtype=torch.int32, device=DEV)
    seen = torch.tensor([2 ** 31 - 3, 2 ** 32 + 9], device=DEV)
    pc.cache_append(made.cache, k, k, made.table, made.lens, starts, seen)
    most = 2 ** 31 - 1
    assert made.cache.pos[made.rows[0][0], 0, :4].tolist() == [most - 2, most - 1, most, most]
    assert made.cache.pos[made.rows[1][0], 0, :4].tolist() == [most] * 4


def test_offsets_of_rows_that_are_not_there():
    """Offsets outside the rows of k and v add no length: only rows that were written count."""
    import paged_cache as pc
    made = Made(920, [3, 5, 0], 2, 64, 16, BF16, room=16)
    k = _randn(921, (6, 2, 64), BF16)
    for starts, new in (([0, 4, 9, 9], [7, 7, 0]), ([0, 2, 6, 20], [5, 9, 0]), ([6, 6, 7, 8], [3, 5, 0]),
                        ([2 ** 31 - 1] * 4, [3, 5, 0]), ([-3, 2, 6, 6], [5, 9, 0])):
        got = pc.cache_append(made.cache, k, k, made.table, made.lens, torch.tensor(starts, device=DEV))
        assert got.tolist() == new, starts
    p = made.rows[0][0]                                       # the last call: rows 0 and 1 behind the three keys
    assert torch.equal(made.cache.k[p, :, 3:5].transpose(0, 1), k[:2])


# --------------------------------------------------------------------------- runs of several units
def _attend_f64(made, q, sm_scale):
    """As paged_ref.attend, in matrix products over a kv head's rows: out, lse, rel (B, H, Q), reach like out, and a
    kv head's weights with the bound of their error: {(b, h): (drawn, tol)}."""
    q4 = (q if q.dim() == 4 else q[:, :, None]).double()
    B, H, Q, D = q4.shape
    c, ps = made.cache, made.ps
    G, n_max = H // c.kv_heads, max(max(made.lens_host), 1)
    out, reach = torch.zeros_like(q4), torch.zeros_like(q4)
    lse = torch.full(q4.shape[:3], float("-inf"), dtype=torch.float64, device=DEV)
    rel, drawn = torch.zeros_like(lse), {}
    for b, n in enumerate(made.lens_host):
        if n == 0:
            continue
        ids = made.table[b, :-(-n // ps)].long()
        ends = (n - (Q - 1) + torch.arange(Q, device=DEV)).repeat(G)              # rows are (head of the group, query)
        unseen = torch.arange(n, device=DEV) >= ends[:, None]
        some = (ends > 0)[:, None]
        for h in range(c.kv_heads):
            k = c.k[ids, h].reshape(-1, D)[:n].double()
            v = c.v[ids, h].reshape(-1, D)[:n].double()
            rows = q4[b, h * G:(h + 1) * G].reshape(-1, D)
            s = (rows @ k.t().contiguous() * sm_scale).masked_fill(unseen, float("-inf"))
            p = torch.where(some, torch.softmax(torch.where(some, s, 0.0), dim=-1), 0.0)
            size = (rows.abs() @ k.abs().t().contiguous() * abs(sm_scale)).masked_fill(unseen, 0.0).amax(dim=-1)
            r = 2 * (D + 8) * U * size + (n_max + 64) * U
            part = slice(h * G, (h + 1) * G)
            out[b, part] = (p @ v).view(G, Q, D)
            reach[b, part] = (p @ v.abs()).view(G, Q, D)
            lse[b, part] = torch.where(some[:, 0], torch.logsumexp(torch.where(some, s, 0.0), dim=-1),
                                       float("-inf")).view(G, Q)
            rel[b, part] = r.view(G, Q)
            # each probability off by its row's rel, their sum over the rows by a rounding each
            drawn[b, h] = p.sum(0), (r[:, None] * p).sum(0) + rows.shape[0] * U * p.sum(0)
    return out, lse, rel, reach, drawn


def _check_attend_f64(made, q, got, lse, weight=None, weight0=None, sm_scale=None):
    out, want_lse, rel, reach, drawn = _attend_f64(made, q, 1 / math.sqrt(q.shape[-1]) if sm_scale is None else sm_scale)
    half, tiny = _half_step(q.dtype), torch.finfo(q.dtype).smallest_normal
    tol = (rel[..., None] * reach + half * out.abs()) * 1.01 + tiny * half
    err = (got.double().reshape(out.shape) - out).abs()
    assert torch.all(err <= tol), f"out: {(err / tol).max().item():.2f} of the bound"
    if lse is not None:
        lse, fine = lse.double().reshape(want_lse.shape), torch.isfinite(want_lse)
        assert torch.equal(torch.isfinite(lse), fine) and torch.all(lse[~fine] == float("-inf"))
        off = (lse - want_lse).abs()[fine] / (rel + 4 * U * (1 + want_lse.abs()))[fine]
        assert torch.all(off <= 1), f"lse: {off.max().item():.2f} of the bound"
    if weight is None:
        return
    grow, bound = weight0.double(), torch.zeros_like(weight0, dtype=torch.float64)
    touched = torch.zeros_like(weight0, dtype=torch.bool)
    for (b, h), (w, t) in drawn.items():
        ids = made.table[b, :-(-len(w) // made.ps)].long()
        pad = len(ids) * made.ps - len(w)
        w, t = (torch.nn.functional.pad(x, (0, pad)).view(-1, made.ps) for x in (w, t))
        grow[ids, h] += w
        bound[ids, h] += t
        touched[ids, h] = (torch.arange(len(ids) * made.ps, device=DEV) < len(ids) * made.ps - pad).view(-1, made.ps)
    # one addition in fp32; a probability below the normal range may go
    tol = bound * 1.01 + 2 * U * grow.abs() + 2.0 ** -120
    off = ((weight.double() - grow).abs() / tol)[touched]
    assert torch.all(off <= 1), f"weight: {off.max().item():.2f} of the bound, {int((off > 1).sum())} keys"
    assert torch.equal(weight[~touched], weight0[~touched]), "a weight outside the sequences changed"


def _ragged(seed, B, low, high):
    """Lengths of low to high with empty and very short sequences among them."""
    g = torch.Generator().manual_seed(seed)
    lens = torch.randint(low, high, (B,), generator=g).tolist()
    for i in range(2, B, 5):
        lens[i] = (0, 1, 33, 0, 127)[i // 5 % 5]
    return lens


RUNS = [
    # B, lengths, H, Hkv, Q, D, page size, dtype: each gives the chip's workgroups three units and more
    (26, (900, 3600), 16, 8, 1, 64, 16, BF16),
    (30, (900, 3600), 8, 8, 1, 128, 64, F16),
    (20, (900, 2100), 8, 8, 1, 64, 32, F32),
    (24, (1200, 3600), 320, 8, 1, 128, 16, F16),               # two row tiles, one query
    (24, (1200, 3600), 512, 8, 1, 64, 16, BF16),               # the same with weights from scores formed again
    (26, (900, 3600), 32, 8, 3, 128, 16, BF16),
    (26, (900, 3600), 16, 8, 7, 64, 8, F16),
    (18, (900, 2200), 16, 8, 5, 128, 16, F32),
    (26, (900, 3600), 32, 8, 16, 128, 32, BF16),               # 64 rows, two tiles of 32
    (26, (900, 3600), 32, 8, 20, 128, 16, BF16),               # 80 rows: keys through LDS
    (26, (900, 3600), 32, 8, 40, 64, 8, F16),                  # 160 rows: two tiles of 128
    (30, (900, 3600), 24, 8, 33, 128, 64, F16),
]


@pytest.mark.parametrize("case", range(len(RUNS)))
def test_attention_in_runs_of_several_units_and_heads(case):
    """Runs that hold several units, that end one kv head and begin the next, or that hold whole ones."""
    import paged_cache as pc
    B, (low, high), H, Hkv, Q, D, ps, dtype = RUNS[case]
    lens = _ragged(case, B, low, high)
    print(f"[case] runs {RUNS[case]}", flush=True)
    unit = 64 if dtype == F32 else 128
    units = Hkv * sum(max(1, -(-max(n - (Q - 1), 0) // unit)) for n in lens)
    assert units >= 3 * (768 if D == 64 and H // Hkv * Q <= 16 else 512), units    # at most as many runs, so three each
    made = Made(1000 + 10 * case, lens, Hkv, D, ps, dtype, layout=("head", "slot", "pair")[case % 3])
    made.cache.weight.zero_()
    if case % 2:                                              # additions to weights that keys have
        made.cache.weight.add_(0.25)
    q = _randn(1001 + 10 * case, (B, H, Q, D) if Q > 1 else (B, H, D), dtype, 1.5)
    weight0 = made.cache.weight.clone()
    plain = pc.paged_attention(q, made.cache, made.table, made.lens)
    got, lse = pc.paged_attention(q, made.cache, made.table, made.lens, accumulate=True, want_lse=True)
    _check_attend_f64(made, q, got, lse, made.cache.weight, weight0)
    assert torch.equal(plain, got)
    before = made.cache.weight.clone()
    made.cache.weight.copy_(weight0)
    again = pc.paged_attention(q, made.cache, made.table, made.lens, accumulate=True)
    assert torch.equal(again, got) and torch.equal(made.cache.weight, before)


WEIGHTS = [
    # lens, H, Hkv, Q, D, page size, dtype
    ([5000, 4097], 8, 2, 1, 128, 64, BF16), ([1000, 0, 257, 511], 32, 8, 1, 128, 16, BF16),
    ([2500], 16, 1, 1, 128, 256, F16), ([3000, 77], 6, 2, 1, 128, 1, F32), ([2513, 90], 71, 1, 1, 64, 8, BF16),
    ([1500, 7], 4, 2, 40, 128, 16, F32), ([4000, 9, 0, 1301], 8, 2, 16, 128, 16, BF16),
    ([6000, 33, 5], 28, 4, 32, 128, 32, F16), ([610, 90], 8, 2, 20, 128, 4, BF16), ([4000, 40], 8, 2, 3, 64, 16, F32),
]


@pytest.mark.parametrize("case", range(len(WEIGHTS)))
def test_weights_of_many_keys(case):
    """What each key draws, from weights of zero: a key of thousands draws little, and all of it counts."""
    import paged_cache as pc
    lens, H, Hkv, Q, D, ps, dtype = WEIGHTS[case]
    print(f"[case] weights {WEIGHTS[case]}", flush=True)
    made = Made(1300 + 10 * case, lens, Hkv, D, ps, dtype)
    made.cache.weight.zero_()
    q = _randn(1301 + 10 * case, (len(lens), H, Q, D), dtype, 1.5)
    weight0 = made.cache.weight.clone()
    got, lse = pc.paged_attention(q, made.cache, made.table, made.lens, accumulate=True, want_lse=True)
    _check_attend_f64(made, q, got, lse, made.cache.weight, weight0)


def test_weights_of_two_streams_at_once():
    import paged_cache as pc
    a, b = Made(1400, [3000, 100], 4, 128, 16, BF16), Made(1420, [700, 2900], 2, 64, 32, F16)
    qa, qb = _randn(1401, (2, 16, 128), BF16), _randn(1421, (2, 16, 40, 64), F16)
    ones = [pc.PagedCache(m.cache.k, m.cache.v, m.cache.weight.clone(), m.cache.pos) for m in (a, b)]
    for _ in range(4):
        pc.paged_attention(qa, ones[0], a.table, a.lens, accumulate=True)
        pc.paged_attention(qb, ones[1], b.table, b.lens, accumulate=True)
    torch.cuda.synchronize()
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(4):
        with torch.cuda.stream(s):
            pc.paged_attention(qa, a.cache, a.table, a.lens, accumulate=True)
        with torch.cuda.stream(t):
            pc.paged_attention(qb, b.cache, b.table, b.lens, accumulate=True)
    torch.cuda.synchronize()
    assert torch.equal(a.cache.weight, ones[0].weight) and torch.equal(b.cache.weight, ones[1].weight)


@pytest.mark.parametrize("D,dtype", [(64, BF16), (128, BF16), (64, F16), (128, F16)])
@pytest.mark.parametrize("Q", [20, 40])
def test_infinite_values_among_many_rows(Q, D, dtype):
    """A workgroup of 128 rows repeats a kv head whose values are infinite, and not the next one of its run."""
    import paged_cache as pc
    inf = float("inf")
    # one page a sequence and kv head of 8, so that a run holds several heads; and one long sequence, cut into runs
    for lens in ([100] * 90 + [0, 33] * 10, [5000, 250]):
        made = Made(1500, lens, 8, D, 128, dtype)
        made.cache.weight.zero_()
        other = made.cache.weight.clone()
        q = _randn(1501, (len(lens), 32, Q, D), dtype)
        clean, lse = pc.paged_attention(q, made.cache, made.table, made.lens, accumulate=True, want_lse=True)
        v, was = made.cache.v, made.cache.v.clone()
        p = made.rows[1][0]
        v[p, 2, 5, 7], v[p, 2, 6, 9], v[p, 2, 7, 9], v[p, 2, 8, 11] = inf, inf, -inf, -inf
        v[made.rows[0][0], 5, 0, 0] = -inf
        marked = pc.PagedCache(made.cache.k, v, other, made.cache.pos)
        got, same = pc.paged_attention(q, marked, made.table, made.lens, accumulate=True, want_lse=True)
        assert torch.all(got[1, 8:12, :, 7] == inf) and torch.isnan(got[1, 8:12, :, 9]).all()
        assert torch.all(got[1, 8:12, :, 11] == -inf) and torch.all(got[0, 20:24, :, 0] == -inf)
        keep = torch.ones_like(got, dtype=torch.bool)
        keep[1, 8:12, :, [7, 9, 11]] = False
        keep[0, 20:24, :, 0] = False
        assert torch.isfinite(got[keep]).all()
        # rows of other kv heads are not repeated in fp32: the same bits; the repeated ones within the bound
        v.copy_(was)
        full = torch.where(keep, got, clean)
        _check_attend_f64(made, q, full, same, other, torch.zeros_like(other))
        _check_attend_f64(made, q, clean, lse, made.cache.weight, torch.zeros_like(other))
        if len(lens) > 2:                                     # whole heads: others' rows see no repeat
            rest = torch.ones(got.shape[:2], dtype=torch.bool, device=DEV)
            rest[1, 8:12] = rest[0, 20:24] = False
            assert torch.equal(got[rest], clean[rest])


# ------------------------------------------------------------------------------ large scores and values
LARGE = [
    # H, Hkv, Q, D, dtype, width of the table in keys
    (8, 2, 1, 64, BF16, 512), (8, 2, 1, 128, F32, 512),       # one launch
    (8, 2, 1, 64, F16, 4096), (8, 2, 1, 128, F32, 4096),      # split
    (40, 1, 1, 64, BF16, 4096), (96, 1, 1, 64, BF16, 4096),   # several row tiles, from stored scores and formed again
    (8, 2, 5, 128, BF16, 4096), (8, 2, 5, 64, F32, 4096), (8, 2, 16, 64, F16, 4096), (8, 2, 20, 128, BF16, 4096),
]


@pytest.mark.parametrize("case", range(len(LARGE)))
def test_weights_at_large_scores(case):
    """Scores that are whole numbers near 1024, with no rounding in them: a weight is off by what its softmax and its sums
    round, not by what a logarithm near 1024 would (2^-14 of it)."""
    import paged_cache as pc
    H, Hkv, Q, D, dtype, width = LARGE[case]
    print(f"[case] large scores {LARGE[case]}", flush=True)
    lens = [50, 37, 51 + Q]
    made = Made(1600, lens, Hkv, D, 16, dtype, extra_width=width // 16 - 6)
    c = made.cache
    c.weight.zero_()
    small = torch.randint(0, 3, c.k.shape, generator=torch.Generator().manual_seed(1601)).to(dtype).to(DEV)
    c.k.zero_()
    c.k[..., 0], c.k[..., 1] = 32.0, small[..., 1]
    q = torch.zeros((3, H, Q, D), dtype=dtype, device=DEV)
    q[..., 0] = 32.0
    q[..., 1] = torch.randint(0, 3, (3, H, Q), generator=torch.Generator().manual_seed(1602)).to(dtype).to(DEV)
    weight0 = c.weight.clone()
    pc.paged_attention(q, c, made.table, made.lens, sm_scale=1.0, accumulate=True)
    _, _, _, _, drawn = _attend_f64(made, q, 1.0)
    for (b, h), (w, _) in drawn.items():
        ids = made.table[b, :-(-len(w) // 16)].long()
        got = c.weight[ids, h].reshape(-1)[:len(w)].double()
        # The differences of scores, down to -4, are whole.  exp: the argument times log2(e), at most 6, rounds by 6 u and
        # log2(e) itself by 4 u in the exponent, and the result by a step; n of them are summed, the sum inverted, the two
        # multiplied and the rows summed; twice the first, for p and its sum, and 16 u for what is left
        n, rows = len(w), H // Hkv * Q
        assert torch.all((got - w).abs() <= (2 * 12 + n + 2 * rows + 16) * U * w), f"{((got - w).abs() / w).max().item():.2e}"
    assert torch.equal(c.weight[made.free], weight0[made.free])


@pytest.mark.parametrize("D,dtype,H,Hkv", [(64, F32, 8, 2), (128, F32, 8, 2), (64, BF16, 8, 2), (128, BF16, 8, 2),
                                           (64, BF16, 40, 1), (128, BF16, 160, 2)])
@pytest.mark.parametrize("Q", [1, 5, 20])
@pytest.mark.parametrize("lens", [[900, 2, 40], [6000, 31, 700]])
def test_attention_of_values_near_the_largest(D, dtype, H, Hkv, Q, lens):
    """A mean of values near the type's largest is finite, however many keys it is of: no sum exceeds it."""
    import paged_cache as pc
    print(f"[case] large values {D} {dtype} {H}/{Hkv} Q={Q} {lens}", flush=True)
    made = Made(1700, lens, Hkv, D, 16, dtype)
    v = made.cache.v
    v[..., 3], v[..., 5] = 3.0e38, -3.0e38
    v[..., 7] = torch.where(v[..., 7].float() > 0, 3.0e38, -3.0e38).to(dtype)
    q = _randn(1701, (len(lens), H, Q, D), dtype)
    got, lse = pc.paged_attention(q, made.cache, made.table, made.lens, want_lse=True)
    assert torch.isfinite(got).all()
    _check_attend_f64(made, q, got, lse)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("Q", [1, 5, 20])
def test_attention_of_small_values(dtype, Q):
    """Values far below 1 keep their precision beside large ones of other dims."""
    import paged_cache as pc
    for lens in ([900, 40], [5000, 200]):
        made = Made(1800, lens, 2, 64, 16, dtype)
        made.cache.v[..., :32] *= 1e-30
        q = _randn(1801, (2, 8, Q, 64), dtype)
        got, lse = pc.paged_attention(q, made.cache, made.table, made.lens, want_lse=True)
        _check_attend_f64(made, q, got, lse)


@pytest.mark.parametrize("case", [0, 2, 5, 7, 8, 9])
def test_large_values_in_runs_of_several_heads(case):
    """Some heads of a run repeat their keys for their large values, the others do not."""
    import paged_cache as pc
    B, (low, high), H, Hkv, Q, D, ps, dtype = RUNS[case]
    lens = _ragged(case, B, low, high)
    print(f"[case] large values in runs {RUNS[case]}", flush=True)
    made = Made(1900 + case, lens, Hkv, D, ps, dtype)
    made.cache.weight.zero_()
    for b in range(0, B, 3):
        for p in made.rows[b]:
            if p >= 0:
                made.cache.v[p, b % Hkv, :, 1:9] = 3.0e38 if b % 2 else -3.0e38
    q = _randn(1901 + case, (B, H, Q, D), dtype, 1.5)
    weight0 = made.cache.weight.clone()
    got, lse = pc.paged_attention(q, made.cache, made.table, made.lens, accumulate=True, want_lse=True)
    assert torch.isfinite(got).all()
    _check_attend_f64(made, q, got, lse, made.cache.weight, weight0)


@pytest.mark.parametrize("H,Hkv,Q,D,dtype", [(16, 8, 1, 64, BF16), (512, 8, 1, 64, F16), (8, 8, 1, 128, F32), (16, 8, 3, 128, BF16),
                                             (32, 8, 16, 64, F16), (32, 8, 20, 128, BF16)])
def test_split_calls_with_weights_in_two_graphs(H, Hkv, Q, D, dtype):
    """Two captured calls, replayed in turn with eager work between them, give the eager call's bits each time."""
    import paged_cache as pc
    print(f"[case] graphs {H}/{Hkv} Q={Q} D={D} {dtype}", flush=True)
    made = [Made(2000 + i, lens, Hkv, D, 16, dtype) for i, lens in enumerate(([3000, 17, 0, 1900], [1200, 2600, 5, 64]))]
    q = [_randn(2010 + i, (4, H, Q, D), dtype) for i in range(2)]
    start = [m.cache.weight.clone() for m in made]

    def call(i):
        return pc.paged_attention(q[i], made[i].cache, made[i].table, made[i].lens, accumulate=True, want_lse=True)
    want = []
    for i in range(2):
        out, lse = call(i)
        want.append((out, lse, made[i].cache.weight.clone()))
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(i))
        graphs.append(g)
    for turn in range(3):
        for i in (turn % 2, 1 - turn % 2):
            made[i].cache.weight.copy_(start[i])
            for x in outs[i]:
                x.fill_(7.0)
            pc.paged_attention(q[1 - i], made[1 - i].cache, made[1 - i].table, made[1 - i].lens)    # eager work
            graphs[i].replay()
            torch.cuda.synchronize()
            for x, w in zip((*outs[i], made[i].cache.weight), want[i]):
                assert torch.equal(x, w), f"replay {turn} of graph {i}"
