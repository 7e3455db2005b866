"""GPU: one plan's norm while its gradients change from call to call -- larger, smaller, zero, one element -- so a partial sum
of a call before would show, in calls enqueued back to back and in a graph."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

EPS32 = 2.0 ** -24
# elements: one workgroup, some, one to a CU, two to a CU
SIZES = [700, 603136, 5_000_003, 70_000_001]


def plan_and_gradients(torch, n, bf16):
    from nerf_amd.api import AdamW
    g = torch.zeros(n, dtype=torch.bfloat16 if bf16 else torch.float32, device="cuda")
    third = n // 3
    parts = [(0, third), (third, 1), (third + 1, n - third - 1)]
    plan = AdamW([dict(g=g.data_ptr() + o * g.element_size(), n=c, g_bf16=bf16) for o, c in parts], state_bits=0)
    return g, plan


def changes(torch, n, bf16):
    """what the gradients become, call by call"""
    gen = torch.Generator(device="cuda").manual_seed(n)
    base = torch.randn(n, device="cuda", generator=gen)
    one = torch.zeros(n, device="cuda")
    one[n - 1] = 3.0
    every = [base * 1e3, base * 1e-3, one, base.abs() + 1, torch.zeros(n, device="cuda"), base * torch.linspace(-1, 1, n, device="cuda"), base.flip(0) * 50]
    return [t.to(torch.bfloat16 if bf16 else torch.float32) for t in every]


def expected(torch, g, div):
    return (g.double().square().sum().sqrt() / div).item()


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("n", SIZES)
def test_norm_of_gradients_that_change(gpu, n, bf16):
    torch = pytest.importorskip("torch")
    g, plan = plan_and_gradients(torch, n, bf16)
    every = changes(torch, n, bf16)
    out = torch.full((4 * len(every),), -1.0, device="cuda")
    torch.cuda.synchronize()
    for turn in range(4):  # the default stream is the library's: no wait between the calls
        for k, x in enumerate(every):
            g.copy_(x)
            plan.grad_norm(out.data_ptr() + 4 * (turn * len(every) + k), 48.0)
    torch.cuda.synchronize()
    got = out.cpu().numpy().reshape(4, -1)
    want = np.array([expected(torch, x, 48.0) for x in every])
    assert (np.abs(got - want) <= 1.001 * EPS32 * want).all(), (got, want)  # sums in 64 bits, one rounding
    plan.destroy()


@pytest.mark.parametrize("n", SIZES[:3])
def test_norm_in_a_graph_of_gradients_that_change(gpu, n):
    """two norms of one plan in a graph, the gradients halved between them, and others in place before every replay"""
    torch = pytest.importorskip("torch")
    from nerf_amd._lib import lib
    g, plan = plan_and_gradients(torch, n, False)
    every = changes(torch, n, False)
    out = torch.zeros(2, device="cuda")
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    try:
        with torch.cuda.graph(graph, stream=side):
            lib.nerf_set_stream(C.c_void_p(side.cuda_stream))
            plan.grad_norm(out.data_ptr(), 2.0)
            g.mul_(0.5)
            plan.grad_norm(out.data_ptr() + 4, 2.0)
    finally:
        lib.nerf_set_stream(None)
    for x in every + every:
        g.copy_(x)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = expected(torch, x, 2.0)
        got = out.cpu().numpy()
        assert abs(got[0] - want) <= 1.001 * EPS32 * want and abs(got[1] - want / 2) <= 1.001 * EPS32 * want / 2
        plan.grad_norm(out.data_ptr())  # eager work between the replays
        torch.cuda.synchronize()
        assert abs(out[0].item() - want) <= 1.001 * EPS32 * want
    plan.destroy()


def test_norm_that_clips_follows_the_gradients(gpu):
    """norm and clipped step, the norm compared with the gradients' and not taken from the device"""
    torch = pytest.importorskip("torch")
    import lowbit_ref as ref
    from nerf_amd.api import AdamW
    n, lr = 50_000, 1e-3
    gen = torch.Generator(device="cuda").manual_seed(1)
    w, m, v = (torch.zeros(n, device="cuda") for _ in range(3))
    g, norm = torch.zeros(n, device="cuda"), torch.zeros(1, device="cuda")
    torch.cuda.synchronize()
    plan = AdamW([dict(w=w.data_ptr(), g=g.data_ptr(), m=m.data_ptr(), v=v.data_ptr(), n=n)])
    for step, size in enumerate((1.0, 100.0, 0.01, 30.0), 1):
        g.normal_(generator=gen).mul_(size)
        before = [t.cpu().numpy() for t in (w, g, m, v)]
        plan.grad_norm(norm.data_ptr(), 1.0)
        plan.step(step, lr, 1.0, norm.data_ptr(), 10.0)
        torch.cuda.synchronize()
        length = np.sqrt((before[1].astype(np.float64) ** 2).sum())
        factor = min(1.0, 10.0 / length)
        w64, m64, v64, _ = ref.adamw_step(before[0], before[1], before[2], before[3], step, lr, 1.0, factor)
        # m: the norm's rounding, the factor's, and five more, relative to its terms; v: twice that
        b1 = float(np.float32(0.9))
        size_m = np.abs(b1 * before[2]) + np.abs(m64 - b1 * before[2])
        assert (np.abs(m.cpu().numpy() - m64) <= 8 * EPS32 * size_m + 1e-44).all()
        assert (np.abs(v.cpu().numpy() - v64) <= 12 * EPS32 * v64 + 1e-44).all()
    plan.destroy()
