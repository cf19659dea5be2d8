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
