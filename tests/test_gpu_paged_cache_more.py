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
