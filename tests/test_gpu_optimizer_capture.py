"""GPU: a plan's calls on the default stream while another, blocking stream is captured, which the runtime answers with an error:
refused as a capture is, and nothing of it is left for the next call to report."""
import ctypes as C

import numpy as np
import pytest

from test_gpu_optimizer import Case

pytestmark = pytest.mark.gpu


def test_calls_beside_another_streams_capture(gpu):
    from nerf_amd._lib import NerfAdamwTensor, lib
    from nerf_amd.api import DeviceArray
    case, norm = Case([5000], 32, 3), DeviceArray.zeros(1)
    before = case.aw.read()[0].copy()
    stream, graph, plan = C.c_void_p(), C.c_void_p(), C.c_void_p()
    table = (NerfAdamwTensor * 1)(NerfAdamwTensor(g=case.ag.ptrs[0], n=5000))
    assert lib.hipStreamCreate(C.byref(stream)) == 0
    assert lib.hipStreamBeginCapture(stream, 0) == 0
    answers = [lib.nerf_adamw_step(case.plan.handle, 1, 1e-3, 1.0, None, 0.0, 0), lib.hipPeekAtLastError(),
               lib.nerf_adamw_create(table, 1, 0, 0.9, 0.999, 1e-8, C.byref(plan)), lib.hipPeekAtLastError()]
    ended = lib.hipStreamEndCapture(stream, C.byref(graph))  # an error where the runtime gave the capture up
    if ended == 0 and graph.value:
        lib.hipGraphDestroy(graph)
    lib.hipGetLastError()
    assert lib.hipStreamDestroy(stream) == 0
    assert answers == [1, 0, 1, 0] and not plan.value
    assert np.array_equal(case.aw.read()[0], before)
    assert lib.nerf_grad_norm(case.plan.handle, 1.0, norm.ptr) == 0
    assert lib.nerf_adamw_step(case.plan.handle, 1, 1e-3, 1.0, None, 0.0, 0) == 0
    want = np.sqrt((case.g[0].astype(np.float64) ** 2).sum())
    assert abs(norm.numpy()[0] - want) <= 1.001 * 2.0 ** -24 * want and not np.array_equal(case.aw.read()[0], before)
