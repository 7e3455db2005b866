"""GPU: products of rows whose values are all small, and of the largest that are allowed.  No part of an input is lost whatever its size, so the bound is the one
of ordinary rows, relative to the sum of magnitudes."""
import numpy as np
import pytest

import lowbit_ref as ref
from product_check import check
from test_gpu_w4 import run, weights

pytestmark = pytest.mark.gpu


def small(m, k, size, seed):
    """values of either sign between size and 8 size, every one an fp32 number"""
    rng = np.random.default_rng(seed)
    x = (size * 2.0 ** rng.uniform(0, 3, (m, k)) * rng.choice([-1.0, 1.0], (m, k))).astype(np.float32)
    assert (x != 0).all()
    return x


def large_weights(n, k, seed):
    rng = np.random.default_rng(seed)
    return (rng.normal(size=(n, k)) * 1e30).astype(np.float32)


SIZES = [1e-33, 1e-34, 1e-35, 1e-36, 1e-37, 1e-38, 1e-39, 1e-40, 1e-42, 1e-44]


@pytest.mark.parametrize("m", [1, 2, 3, 6, 20, 40])
@pytest.mark.parametrize("size,bf16", [(s, False) for s in SIZES] + [(s, True) for s in SIZES if s > 2.0 ** -133])
def test_rows_of_small_values(gpu, size, bf16, m):
    n, k = 37, 200
    codes, scales = ref.quantize_w4(large_weights(n, k, 3), 32)
    w = ref.dequantize_w4(codes, scales, k, 32)
    held = ref.bf16(small(m, k, size, m)) if bf16 else small(m, k, size, m)
    x = ref.from_bf16(held) if bf16 else held
    got = run(held, codes, scales, 32, n, k, bf16, False, 0)
    check(got, x.astype(np.float64), w, False, 0)


# several slices, parts and launches' shapes, rows and columns that fill no tile, a last column inside eight
SHAPES = [(3, 35, 20000), (4, 9000, 5000), (16, 16, 16384), (17, 65, 257), (20, 40, 5000), (24, 300, 1001), (33, 17000, 700), (64, 256, 512),
          (64, 8300, 1100), (65, 70, 96), (200, 300, 260)]


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
def test_small_values_in_every_shape(gpu, shape, group):
    """rows from 1e-44 to 1e-33: the smallest decide their own row's bound"""
    m, n, k = shape
    codes, scales = ref.quantize_w4(large_weights(n, k, 3), group)
    w = ref.dequantize_w4(codes, scales, k, group)
    x = np.concatenate([small(1, k, 10.0 ** (-44 + 11 * (i % 7) / 6), i) for i in range(m)])
    check(run(x, codes, scales, group, n, k, False, False, 0), x.astype(np.float64), w, False, 0)


@pytest.mark.parametrize("m", [1, 2, 3, 20, 40])
@pytest.mark.parametrize("spread", [1.0, 3e5], ids=["beside each other", "scales over many powers of two"])
def test_small_values_beside_large_ones_that_meet_zeros(gpu, m, spread):
    """a row's largest values multiply zeros: what is left is decided by its smallest ones"""
    n, k, group = 45, 700, 64
    w = large_weights(n, k, 5) * np.float32(spread) ** np.linspace(-1, 1, n, dtype=np.float32)[:, None]
    w[:, 128:512] = 0.0
    codes, scales = ref.quantize_w4(w, group)
    w = ref.dequantize_w4(codes, scales, k, group)
    x = small(m, k, 1e-38, m)
    x[:, 128:512] = small(m, 384, 1e20, m + 1)
    got = run(x, codes, scales, group, n, k, False, False, 0)
    x[:, 128:512] = 0.0  # they add nothing, and nothing to the bound
    check(got, x.astype(np.float64), w, False, 0)


@pytest.mark.parametrize("m", [3, 20, 70])
def test_small_values_leave_other_rows_alone(gpu, m):
    """the bits of ordinary rows are the same whether a row of small values, an infinity or a NaN is beside them"""
    n, k, group = 90, 1030, 32
    codes, scales = ref.quantize_w4(weights(n, k, 6), group)
    rng = np.random.default_rng(m)
    x = rng.normal(size=(m, k)).astype(np.float32)
    plain = run(x, codes, scales, group, n, k, False, False, 0)
    x[1] = small(1, k, 1e-40, 2)
    x[2, 7], x[2, 1029] = np.inf, 1e-41
    mixed = run(x, codes, scales, group, n, k, False, False, 0)
    rest = [i for i in range(m) if i not in (1, 2)]
    assert np.array_equal(plain[rest], mixed[rest])
    w = ref.dequantize_w4(codes, scales, k, group)
    with np.errstate(all="ignore"):
        want = np.array([(x[2].astype(np.float64) * w[j]).sum() for j in range(n)])
    assert np.array_equal(np.isnan(mixed[2]), np.isnan(want)) and np.array_equal(mixed[2][np.isinf(want)], want[np.isinf(want)])
    assert not np.isfinite(mixed[2]).any() and np.isfinite(mixed[1]).all()


@pytest.mark.parametrize("m", [3, 40])
def test_small_values_with_scales_that_are_small_too(gpu, m):
    """products below the smallest fp32 number are zero, and others beside them right"""
    n, k, group = 20, 300, 32
    w = np.random.default_rng(7).normal(size=(n, k)).astype(np.float32)
    w[::2] *= np.float32(1e-36)
    w[1::2] *= np.float32(1e36)
    codes, scales = ref.quantize_w4(w, group)
    x = small(m, k, 1e-41, m)
    got = run(x, codes, scales, group, n, k, False, False, 0)
    assert (got[:, ::2] == 0).all()
    check(got[:, 1::2], x.astype(np.float64), ref.dequantize_w4(codes, scales, k, group)[1::2], False, 0)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("m", [1, 2, 3, 20, 64])
def test_rows_of_the_largest_values(gpu, m, group, bf16):
    """all of one sign and just below 2^118, against the largest code: the sum of a group of 128 is below 2^128"""
    n, k = 20, 300
    w = np.random.default_rng(4).uniform(5.5e-6, 6e-6, (n, k)).astype(np.float32)
    codes, scales = ref.quantize_w4(w, group)
    w = ref.dequantize_w4(codes, scales, k, group)
    x = np.random.default_rng(m).uniform(0.9, 0.99, (m, k)).astype(np.float32) * np.float32(2.0 ** 118)
    held = ref.bf16(x) if bf16 else x
    x = ref.from_bf16(held) if bf16 else x
    check(run(held, codes, scales, group, n, k, bf16, False, 0), x.astype(np.float64), w, False, 0)


def test_dequantize_of_the_largest_weights(gpu):
    """6 times a bf16 scale is an fp32 number up to 255 / 256 of 2^128: 3.38e38 comes back, fp32's largest as an infinity"""
    from nerf_amd._lib import lib
    from nerf_amd.api import DeviceArray
    w = np.zeros((2, 32), np.float32)
    w[0, :3] = [3.38e38, -3.38e38, 1e38]
    w[1, :2] = np.finfo(np.float32).max
    d, codes, scales, back = DeviceArray.from_numpy(w), DeviceArray((2, 16), np.uint8), DeviceArray((2, 1), np.uint16), DeviceArray((2, 32))
    assert lib.nerf_quantize_w4(d.ptr, 32, 2, 32, 32, codes.ptr, scales.ptr) == 0
    assert lib.nerf_dequantize_w4(codes.ptr, scales.ptr, 2, 32, 32, back.ptr, 32) == 0
    got, want = back.numpy(), ref.dequantize_w4(codes.numpy(), scales.numpy(), 32, 32)
    assert np.array_equal(got[0].astype(np.float64), want[0]) and np.isfinite(got[0]).all()
    assert np.isposinf(got[1, :2]).all() and (want[1, :2] > np.finfo(np.float32).max).all()
