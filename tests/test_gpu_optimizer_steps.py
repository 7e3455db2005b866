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


@pytest.mark.parametrize("bf16", [False, True])
def test_states_in_8_bits_follow_64_bit_ones_where_a_seed_rounds_by_chance(gpu, bf16):
    """300 steps of steady gradients.  Rounding by chance is right on average; what a step adds to the variance of sqrt(v) is at
    most a step of the code (1/16 of the value at most) times the mean change, 0.97 / 2 thousandths of the value and up to
    1 / 2t in the first t steps, and v forgets a thousandth a step: at most 6 % of v, 3 % of its root, and the mean of 4096
    roots that scatter by 12 % is 0.2 % off.  To nearest, where no change is as large as half a step, the mean falls below 0.8."""
    torch = pytest.importorskip("torch")
    from nerf_amd._lib import lib
    from nerf_amd.api import AdamW
    n, lr = 4096, 1e-3
    blocks = lib.nerf_adamw_state_blocks(n)
    new = lambda count, t: torch.zeros(count, dtype=t, device="cuda")  # noqa: E731
    ratio = {}
    for seed in (0, 17):
        gen = torch.Generator(device="cuda").manual_seed(9)
        w, g = new(n, torch.float32), new(n, torch.bfloat16 if bf16 else torch.float32)
        m, v, me, ve = new(n, torch.uint8), new(n, torch.uint8), new(blocks, torch.uint8), new(blocks, torch.uint8)
        right, roots = new(n, torch.float64), new(n, torch.bfloat16)
        torch.cuda.synchronize()
        plan = AdamW([dict(w=w.data_ptr(), g=g.data_ptr(), m=m.data_ptr(), v=v.data_ptr(), m_exp=me.data_ptr(), v_exp=ve.data_ptr(), n=n,
                           g_bf16=bf16)], state_bits=8)
        b2 = float(np.float32(0.999))
        for step in range(1, 301):
            g.copy_(torch.randn(n, device="cuda", generator=gen) * 1e-3)
            plan.step(step, lr, seed=seed)
            right.mul_(b2).add_(g.double().square(), alpha=1 - b2)
        plan.read_states(None, roots.data_ptr())
        torch.cuda.synchronize()
        ratio[seed] = (roots.double() / right.sqrt()).mean().item()
        plan.destroy()
    assert abs(ratio[17] - 1) <= 0.032, ratio
    assert ratio[0] < 0.8, ratio  # what the documentation warns of


def test_a_step_without_a_seed_warns(gpu):
    import warnings
    small, large = Case([300], 8, 5), Case([300], 32, 5)
    with pytest.warns(UserWarning, match="seed"):
        small.plan.step(1, 1e-3)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        small.plan.step(2, 1e-3, seed=0)
        small.plan.step(3, 1e-3, seed=4)
        large.plan.step(1, 1e-3)


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


def test_training_goes_on_bit_for_bit_from_states_that_were_copied_out(gpu):
    """what a checkpoint of an outside plan has to hold: weights, codes, exponents, the step number and the seed"""
    sizes = [700, 5000]
    rng = np.random.default_rng(3)
    gradients = [[rng.normal(0, 1e-2, n).astype(np.float32) for n in sizes] for _ in range(6)]

    def steps(case, first, last):
        for step in range(first, last):
            flat = case.ag.dev.numpy()
            flat[case.ag.start:case.ag.start + sum(sizes)] = np.concatenate(gradients[step - 1])
            case.ag.dev.upload(flat)
            case.plan.step(step, 1e-3, seed=5)

    one, two = Case(sizes, 8, 31), Case(sizes, 8, 32)  # two starts with other contents
    steps(one, 1, 4)
    arenas = lambda case: (case.aw, case.am, case.av, case.ame, case.ave)  # noqa: E731
    for a, b in zip(arenas(one), arenas(two)):
        b.dev.upload(a.dev.numpy())
    steps(one, 4, 7)
    steps(two, 4, 7)
    for a, b in zip(arenas(one), arenas(two)):
        assert np.array_equal(a.dev.numpy(), b.dev.numpy())
