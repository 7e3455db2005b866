"""CPU: a workspace of nerf_gemm_w4 that is sized for the largest batch serves every smaller one."""
import pytest

SHAPES = [(512, 512), (4096, 4096), (8192, 16384), (16384, 8192), (4100, 4090), (16, 16384), (100000, 64), (3, 40000), (1, 1), (5000, 129), (256, 1 << 20)]
ROWS = [*range(1, 140), 200, 256, 300, 511, 512, 1000, 2048, 4000, 8192, 10000, 100000]


@pytest.mark.parametrize("n,k", SHAPES)
def test_more_rows_never_need_less(n, k):
    from nerf_amd._lib import lib
    need = [lib.nerf_gemm_w4_workspace(m, n, k) for m in ROWS]
    assert need == sorted(need)
    assert need[0] == need[1] == 0  # one and two rows need none
    assert need[-1] <= 1 << 24


@pytest.mark.parametrize("n,k", SHAPES[:8])
def test_the_largest_batchs_workspace_is_taken_for_every_smaller_one(n, k):
    """what passes the checks fails with 2 where there is no GPU"""
    from nerf_amd._lib import lib
    if lib.nerf_device_count():
        pytest.skip("the addresses are no GPU's")
    for most in (3, 24, 64, 128, 300):
        size = lib.nerf_gemm_w4_workspace(most, n, k)
        for m in range(1, most + 1):
            rc = lib.nerf_gemm_w4(0x1000, 0, k, 0x2000, 0x3000, 64, 0x4000, 0, n, m, n, k, 0, 0x8000 if size else None, size)
            assert rc == 2, (most, m)
