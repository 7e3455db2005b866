"""GPU: 8-bit states over several steps -- a second moment that overflows, and states that follow 64-bit ones for hundreds of
steps where a seed rounds by chance."""
import numpy as np
import pytest

import lowbit_ref as ref
from test_gpu_optimizer import Arena, Case, check_weights

pytestmark = pytest.mark.gpu


def set_gradients(case, g):
    flat = case.ag.dev.numpy()
    flat[case.ag.start:case.ag.start + len(g)] = g
    case.ag.dev.upload(flat)
    case.g = [g]


def spikes(n):
    """ordinary gradients, and some whose square is not finite, alone in a block and beside each other"""
    g = np.random.default_rng(0).normal(0, 1e-3, n).astype(np.float32)
    g[[5, 300, 301, 700]] = np.float32([1e21, -3e38, 1e30, -2e21])
    return g


@pytest.mark.parametrize("seed", [0, 11])
def test_a_second_moment_that_overflows_does_not_throw_the_weight_away(gpu, seed):
    """One step with gradients of 1e21 and more, then ordinary ones.  With 32-bit states v stays infinite and the weight holds
    still.  In 8 bits both moments start again from zero; from there |m| / sqrt(v) is at most (1 - b1) / sqrt((1 - b2)(1 - b1^2 / b2))
    = 7.3 by Cauchy and Schwarz, and a rounding of m by one step of 1/8 up and of sqrt(v) by one of 1/16 down for each of six
    steps makes that at most 7.3 * (1.125 / 0.9375)^6 = 21.8.  The bias correction is at most 0.24 from step 3 on."""
    n, lr = 1000, 1e-3
    small, large = Case([n], 8, 21), Case([n], 32, 21)
    rng = np.random.default_rng(1)
    gradients = [spikes(n)] + [rng.normal(0, 1e-3, n).astype(np.float32) for _ in range(6)]
    hit = np.array([5, 300, 301, 700])
    for step, g in enumerate(gradients, 2):
        for case in (small, large):
            set_gradients(case, g)
            case.plan.step(step, lr, seed=seed)
    a, b = small.aw.read()[0], large.aw.read()[0]
    assert np.isfinite(a).all()
    assert (np.abs(a - b)[hit] <= 6 * 0.24 * 21.8 * lr + 1e-6).all(), (a[hit], b[hit])


@pytest.mark.parametrize("seed", [0, 11])
def test_a_first_moment_beside_a_root_held_as_zero_counts_as_zero(gpu, seed):
    """the step after, bit for bit, and the values that are read"""
    n = 1000
    case = Case([n], 8, 22, gradient=lambda g: g[0].__setitem__(slice(None), spikes(n)))
    case.plan.step(2, 1e-3, seed=seed)
    w, m, me, v, ve = (x.read()[0] for x in (case.aw, case.am, case.ame, case.av, case.ave))
    gone = v == 0
    assert gone[[5, 300, 301, 700]].all() and gone.sum() == 4 and (m[gone] & 127 > 0).any()
    held = np.where(gone, 0, ref.decode_m(m.astype(np.int64), me)).astype(np.float32)
    out = Arena([np.zeros(n)], np.uint16, 1)
    case.plan.read_states(out.ptrs[0], None)
    assert np.array_equal(ref.from_bf16(out.read()[0]), held)
    g = np.random.default_rng(2).normal(0, 1e-3, n).astype(np.float32)
    set_gradients(case, g)
    case.plan.step(3, 1e-3, seed=seed)
    roots = ref.decode(v, 4, ve).astype(np.float32)
    _, m32, _, r32 = ref.adamw_step(w, g, held, roots, 3, 1e-3, 1.0, root=True, dtype=np.float32)
    share_m, share_r = ref.noise(n, seed, 3, 0)
    assert np.array_equal(case.am.read()[0], ref.encode_m(m32, share_m)[0]) and np.array_equal(case.av.read()[0], ref.encode_r(r32, share_r)[0])
    # check_weights' bound: alpha holds 1 - beta2^3 = 0.003, which loses half a step of beta2^3
    case.w, case.m, case.v = [w], [held], [roots]
    check_weights(case, case.aw.read(), 3, 1e-3, 1.0, 1.0)


def test_a_norm_that_is_not_aligned_is_refused(gpu):
    """a scalar load would read the float before it"""
    from nerf_amd._lib import lib
    from nerf_amd.api import DeviceArray
    case, norm = Case([100], 32, 1), DeviceArray.from_numpy(np.array([1.0, 2.0], np.float32))
    before = case.aw.read()[0].copy()
    for shift in (1, 2, 3):
        assert lib.nerf_adamw_step(case.plan.handle, 1, 1e-3, 1.0, norm.ptr + shift, 1.0, 0) == 1
    assert np.array_equal(case.aw.read()[0], before)
    assert lib.nerf_adamw_step(case.plan.handle, 1, 1e-3, 1.0, norm.ptr + 4, 1.0, 0) == 0
