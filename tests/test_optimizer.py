"""CPU: the low-bit formats' plain statement against itself, and what nerf_adamw_create refuses before it touches
a device (status 1; a list it accepts fails with 2 where there is no GPU)."""
import ctypes as C

import numpy as np
import pytest

import lowbit_ref as ref


def test_codes_round_by_at_most_half_a_step():
    rng = np.random.default_rng(0)
    m = (rng.normal(size=5000) * 10.0 ** rng.uniform(-6, 0, 5000)).astype(np.float32)
    share, _ = ref.noise(len(m), 0, 1, 0)
    for bits, x, (code, exps), back in ((3, m, ref.encode_m(m, share), ref.decode_m), (4, np.abs(m), ref.encode_r(np.abs(m), share),
                                                                                    lambda c, e: ref.decode(c, 4, e))):
        got = back(code, exps)
        top = 2.0 ** (np.repeat(exps.astype(float), ref.BLOCK)[: len(x)] - 127)
        # to nearest: half a step of the value's binade, or of the lowest one; sqrt(v) keeps at least one step
        low = top * 2.0 ** (-14 - bits)
        bound = np.maximum(np.abs(x) * 2.0 ** (-bits - 1), low if bits == 4 else low / 2)
        assert (np.abs(got - x) <= bound).all()
        assert ((np.abs(x) < low / 2) | (np.sign(got) == np.sign(x))).all()
        # a value that a code stands for is its own code, whatever the noise
        again = ref.encode(np.abs(got).astype(np.float32), bits, exps, np.full(len(x), 65535))
        assert (again == (code & 127 if bits == 3 else code)).all()


def test_stochastic_rounding_has_no_bias():
    x = np.full(1 << 16, 1.03, np.float32)
    x[0::ref.BLOCK] = 1.5
    a, b = ref.noise(len(x), 9, 4, 2)
    for code, back in ((ref.encode_m(x, a), ref.decode_m), (ref.encode_r(x, b), lambda c, e: ref.decode(c, 4, e))):
        got = back(*code)[x < 1.4]
        # a mean of n independent roundings with steps s <= 1/8 is off by some s / sqrt(n): five of those
        assert abs(got.mean() - np.float32(1.03)) <= 5 * 0.125 / np.sqrt(len(got))


def _tensor(**kw):
    from nerf_amd._lib import NerfAdamwTensor
    t = dict(w=0x10000, g=0x20000, m=0x30000, v=0x40000, m_exp=0x50000, v_exp=0x60000, w_bf16=0, n=1000, grad_type=0,
             lr_scale=1.0, weight_decay=0.01)
    t.update(kw)
    return NerfAdamwTensor(**t)


def _create(tensors, bits=32, beta1=0.9, beta2=0.999, eps=1e-8, count=None):
    from nerf_amd._lib import NerfAdamwTensor, lib
    out = C.c_void_p(1)
    table = (NerfAdamwTensor * max(1, len(tensors)))(*tensors)
    rc = lib.nerf_adamw_create(table, len(tensors) if count is None else count, bits, beta1, beta2, eps, C.byref(out))
    assert not out.value
    return rc


BAD = {
    "no tensors": ([], {}),
    "state bits": ([_tensor], {"bits": 16}),
    "beta1": ([_tensor], {"beta1": 1.0}),
    "beta2": ([_tensor], {"beta2": -0.1}),
    "beta nan": ([_tensor], {"beta1": float("nan")}),
    "eps": ([_tensor], {"eps": 0.0}),
    "no gradient": ([lambda: _tensor(g=0)], {}),
    "no gradient, norms only": ([lambda: _tensor(g=0)], {"bits": 0}),
    "no weights": ([lambda: _tensor(w=0)], {}),
    "no exponents": ([lambda: _tensor(v_exp=0)], {"bits": 8}),
    "gradient type": ([lambda: _tensor(grad_type=2)], {}),
    "float alignment": ([lambda: _tensor(m=0x30002)], {}),
    "bf16 alignment": ([lambda: _tensor(g=0x20001, grad_type=1)], {}),
    "copy alignment": ([lambda: _tensor(w_bf16=0x70001)], {}),
    "too long": ([lambda: _tensor(n=(1 << 40) + 1)], {}),
    "negative decay": ([lambda: _tensor(weight_decay=-1.0)], {}),
    "lr scale nan": ([lambda: _tensor(lr_scale=float("nan"))], {}),
    "the same tensor twice": ([_tensor, _tensor], {}),
    "states overlap": ([lambda: _tensor(v=0x30000 + 3996)], {}),
    "gradient inside weights": ([lambda: _tensor(g=0x10000 + 1000)], {}),
    "codes overlap": ([lambda: _tensor(v=0x30000 + 999)], {"bits": 8}),
    "exponents overlap": ([lambda: _tensor(v_exp=0x50003)], {"bits": 8}),
}


@pytest.mark.parametrize("name", BAD)
def test_create_refuses(name):
    make, kw = BAD[name]
    assert _create([m() for m in make], **kw) == 1


def test_create_takes_what_is_not_refused():
    """these lists pass the checks: the pointers are no device's, so 1 (a GPU says so) or 2 (there is none)"""
    from nerf_amd._lib import lib
    want = 1 if lib.nerf_device_count() else 2
    ok = [_tensor(n=1000), _tensor(w=0x110000, m=0x130000, v=0x140000, n=1000)]  # one gradient for both
    assert _create(ok) == want
    assert _create([_tensor(v=0x30000 + 1000, v_exp=0x50004)], bits=8) == want
    assert _create([_tensor(w=0, m=0, v=0)], bits=0) == want


def test_calls_on_no_plan_are_refused():
    from nerf_amd._lib import lib
    assert lib.nerf_adamw_step(None, 1, 0.1, 1.0, None, 0.0, 0) == 1
    assert lib.nerf_grad_norm(None, 1.0, 16) == 1
    assert lib.nerf_adamw_read_states(None, 16, 16) == 1
    lib.nerf_adamw_destroy(None)
    assert lib.nerf_adamw_create(None, 1, 32, 0.9, 0.999, 1e-8, C.byref(C.c_void_p())) == 1
    assert [lib.nerf_adamw_state_blocks(n) for n in (0, 1, 256, 257)] == [0, 1, 1, 2]
