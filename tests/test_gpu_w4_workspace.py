"""GPU: one workspace, sized for the largest batch, for every smaller one in turn."""
import numpy as np
import pytest

import lowbit_ref as ref
from product_check import check
from test_gpu_w4 import Guarded, weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,k", [(300, 5000), (4100, 1030)])
def test_one_workspace_for_every_number_of_rows(gpu, n, k):
    from nerf_amd._lib import lib
    from nerf_amd.api import DeviceArray
    codes, scales = ref.quantize_w4(weights(n, k, 2), 64)
    w = ref.dequantize_w4(codes, scales, k, 64)
    most = 130
    x = np.random.default_rng(n).normal(size=(most, k)).astype(np.float32)
    d_c, d_s, d_x = DeviceArray.from_numpy(codes), DeviceArray.from_numpy(scales), DeviceArray.from_numpy(x)
    size = lib.nerf_gemm_w4_workspace(most, n, k)
    ws = Guarded(np.frombuffer(b"\xff" * size, np.uint8))
    for m in [*range(1, 40), 47, 48, 49, 63, 64, 65, 100, most]:
        y = Guarded(np.full((m, n), np.nan, np.float32))
        assert lib.nerf_gemm_w4(d_x.ptr, 0, k, d_c.ptr, d_s.ptr, 64, y.ptr, 0, n, m, n, k, 0, ws.ptr, size) == 0
        check(y.read(), x[:m].astype(np.float64), w, False, 0)
    ws.read()
