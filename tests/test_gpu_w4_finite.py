"""GPU: the products of test_gpu_w4 with a check that a NaN fails.  Gaps between rows of X, an untouched workspace and rows
past the end hold NaN there, so a read of any of them shows."""
import numpy as np
import pytest

import lowbit_ref as ref
import test_gpu_w4 as products
from product_check import check

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def strict(monkeypatch):
    monkeypatch.setattr(products, "check", check)


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("shape", products.SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("bf16", [False, True])
def test_product(gpu, shape, group, bf16):
    products.test_product(gpu, shape, group, bf16)


@pytest.mark.parametrize("x_bf16,y_bf16", [(False, True), (True, False), (False, False), (True, True)])
@pytest.mark.parametrize("m", [1, 2, 7, 16, 40, 80])
def test_product_strides_types_and_swish(gpu, m, x_bf16, y_bf16):
    products.test_product_strides_types_and_swish(gpu, m, x_bf16, y_bf16)


@pytest.mark.parametrize("m", [1, 2, 5, 20])
def test_product_keeps_the_precision_of_fp32(gpu, m):
    products.test_product_keeps_the_precision_of_fp32(gpu, m)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("m", [1, 2, 3, 20])
def test_product_of_subnormal_inputs(gpu, m, bf16):
    products.test_product_of_subnormal_inputs(gpu, m, bf16)


def test_more_rows_than_a_launch_takes(gpu):
    products.test_more_rows_than_a_launch_takes(gpu)


def test_trained_with_8_bit_states_and_answered_in_4_bits(gpu):
    products.test_trained_with_8_bit_states_and_answered_in_4_bits(gpu)


def test_codes_past_four_gib(gpu):
    """rows of W behind 2^32 bytes of codes, Y and the workspace full of NaN before each call; every value of Y is written"""
    torch = pytest.importorskip("torch")
    from nerf_amd._lib import lib
    n, k, group = 66000, 131072, 128
    gen = torch.Generator(device="cuda").manual_seed(3)
    codes = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device="cuda", generator=gen)
    scales = torch.randint(0x3C00, 0x4000, (n, k // group), dtype=torch.int16, device="cuda", generator=gen)
    rows = [0, 1000, 65535, 65536, 65999]
    w = ref.dequantize_w4(codes[rows].cpu().numpy(), scales[rows].cpu().numpy().view(np.uint16), k, group)
    for m in (1, 3, 20):
        x = torch.randn(m, k, device="cuda", generator=gen)
        y = torch.full((m, n), float("nan"), device="cuda")
        size = lib.nerf_gemm_w4_workspace(m, n, k)
        ws = torch.full((size // 4 + 4,), float("nan"), device="cuda")
        torch.cuda.synchronize()
        assert lib.nerf_gemm_w4(x.data_ptr(), 0, k, codes.data_ptr(), scales.data_ptr(), group, y.data_ptr(), 0, n, m, n, k, 0,
                                ws.data_ptr(), size) == 0
        torch.cuda.synchronize()
        assert bool(torch.isfinite(y).all())
        check(y[:, rows].cpu().numpy(), x.cpu().numpy().astype(np.float64), w, False, 0)
    del codes, scales, x, y, ws
    torch.cuda.empty_cache()
