"""GPU: weights in 4 bits -- quantize and dequantize bit for bit against numpy, products against float64."""
import numpy as np
import pytest

import lowbit_ref as ref

pytestmark = pytest.mark.gpu

EPS32 = 2.0 ** -24
GUARD = 64


class Guarded:
    """a device array between guard elements; `shift` elements behind an aligned start"""

    def __init__(self, a, shift=0):
        from nerf_amd.api import DeviceArray
        a = np.ascontiguousarray(a)
        self.shape, self.dtype, self.size, self.start = a.shape, a.dtype, a.size, GUARD + shift
        flat = np.frombuffer(b"\x5a" * (a.itemsize * (a.size + 2 * GUARD + shift)), a.dtype).copy()
        flat[self.start:self.start + a.size] = a.reshape(-1)
        self.dev = DeviceArray.from_numpy(flat)
        self.ptr = self.dev.ptr + self.start * a.itemsize

    def read(self):
        flat = self.dev.numpy()
        out = flat[self.start:self.start + self.size].copy()
        flat[self.start:self.start + self.size] = np.frombuffer(b"\x5a" * flat.itemsize, flat.dtype)[0]
        assert (flat.view(np.uint8) == 0x5A).all(), "guard elements were written"
        return out.reshape(self.shape)


def weights(n, k, seed):
    rng = np.random.default_rng(seed)
    w = (rng.normal(size=(n, k)) * 10.0 ** rng.uniform(-2, 2, (n, 1))).astype(np.float32)
    w[n // 2, :] = 0.0
    return w


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,k", [(1, 1), (3, 31), (5, 32), (4, 33), (17, 150), (512, 512), (9, 127), (33, 129), (2, 4090), (1000, 64), (64, 16384)])
def test_quantize_and_back(gpu, n, k, group):
    from nerf_amd._lib import lib
    w = weights(n, k, n * 7 + k)
    ld = k + 3
    src = np.full((n, ld), np.nan, np.float32)  # what lies between the rows is not read
    src[:, :k] = w
    d = Guarded(src)
    codes, scales = Guarded(np.zeros((n, ref.w4_row_bytes(k)), np.uint8)), Guarded(np.zeros((n, -(-k // group)), np.uint16), 1)
    assert lib.nerf_quantize_w4(d.ptr, ld, n, k, group, codes.ptr, scales.ptr) == 0
    want_codes, want_scales = ref.quantize_w4(w, group)
    assert np.array_equal(scales.read(), want_scales) and np.array_equal(codes.read(), want_codes)
    back = Guarded(np.full((n, ld), 7.0, np.float32), 1)
    assert lib.nerf_dequantize_w4(codes.ptr, scales.ptr, n, k, group, back.ptr, ld) == 0
    got = back.read()
    assert np.array_equal(got[:, :k].astype(np.float64), ref.dequantize_w4(want_codes, want_scales, k, group)) and (got[:, k:] == 7.0).all()


def test_quantize_extremes(gpu):
    """ties, the largest and smallest numbers, and a group that holds a weight that is not finite"""
    from nerf_amd._lib import lib
    w = np.zeros((6, 64), np.float32)
    w[0, :9] = [6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -2.5]
    w[1, :] = np.linspace(-3.4e38, 3.4e38, 64)
    w[2, :] = np.arange(64) * 1e-45
    w[3, 3], w[3, 40] = np.nan, 1.0
    w[4, 3], w[4, 40] = -np.inf, 1.0
    w[5, :] = -0.0
    d, codes, scales = Guarded(w), Guarded(np.zeros((6, 32), np.uint8)), Guarded(np.zeros((6, 2), np.uint16))
    assert lib.nerf_quantize_w4(d.ptr, 64, 6, 64, 32, codes.ptr, scales.ptr) == 0
    want_codes, want_scales = ref.quantize_w4(w, 32)
    assert np.array_equal(scales.read(), want_scales)
    fine = np.ones((6, 2), bool)
    fine[3, 0] = fine[4, 0] = False
    got = codes.read().reshape(6, 2, 16)
    assert np.array_equal(got[fine], want_codes.reshape(6, 2, 16)[fine])
    assert np.isnan(ref.from_bf16(scales.read())[~fine]).all() and np.isfinite(ref.from_bf16(scales.read())[fine]).all()


@pytest.mark.parametrize("power", [-133, -126, -40, 0, 60, 125])
def test_quantize_next_to_borders(gpu, power):
    """every scale mantissa of 8 bits, and weights on each border between codes and up to three fp32 numbers beside it"""
    from nerf_amd._lib import lib
    bits = np.arange(128, 256, dtype=np.float64) * 2.0 ** (power - 7)
    scale = ref.from_bf16((bits.astype(np.float32).view(np.uint32) >> 16).astype(np.uint16)).astype(np.float32)  # cut where subnormal
    borders = np.float32([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    rows = []
    for s in scale:
        if 6.0 * float(s) > 3.4e38:
            continue
        at = (borders * s).astype(np.float32)  # exact, but for subnormal scales: numbers like others there
        w = [s * np.float32(6)] + [v for b in at for v in (b, -b)]
        for b in at:
            up = down = b
            for _ in range(3):
                up, down = np.nextafter(up, np.float32(np.inf)), np.nextafter(down, np.float32(0))
                w += [up, -down, -up, down]
        rows.append(np.float32(w + [0.0] * (-len(w) % 128)))
    w = np.stack(rows)
    n, k = w.shape
    assert k == 128
    d, codes, scales = Guarded(w), Guarded(np.zeros((n, 64), np.uint8)), Guarded(np.zeros((n, 1), np.uint16))
    assert lib.nerf_quantize_w4(d.ptr, k, n, k, 128, codes.ptr, scales.ptr) == 0
    want_codes, want_scales = ref.quantize_w4(w, 128)
    assert np.array_equal(scales.read(), want_scales) and np.array_equal(codes.read(), want_codes)


def run(x, codes, scales, group, n, k, x_bf16, y_bf16, epilogue, ldx=None, ldy=None, shift=0):
    from nerf_amd._lib import lib
    from nerf_amd.api import DeviceArray
    m = x.shape[0]
    ldx, ldy = ldx or k, ldy or n
    xs = np.full((m, ldx), 0x7FC0 if x_bf16 else np.nan, np.uint16 if x_bf16 else np.float32)  # gaps are not read
    xs[:, :k] = x
    d_x, d_c, d_s = Guarded(xs, shift), Guarded(codes), Guarded(scales, shift)
    y = Guarded(np.full((m, ldy), 9, np.uint16 if y_bf16 else np.float32), shift)
    size = lib.nerf_gemm_w4_workspace(m, n, k)
    ws = Guarded(np.frombuffer(b"\xff" * size, np.uint8)) if size else None  # not cleared: NaN where it is read unwritten
    assert lib.nerf_gemm_w4(d_x.ptr, int(x_bf16), ldx, d_c.ptr, d_s.ptr, group, y.ptr, int(y_bf16), ldy, m, n, k, epilogue,
                            ws.ptr if ws else None, size) == 0
    got = y.read()
    if ws:
        ws.read()
    assert (got[:, n:] == 9).all()
    got = got[:, :n]
    return ref.from_bf16(got) if y_bf16 else got


def check(got, x, w, y_bf16, epilogue):
    """Products are exact.  A sum of K terms in chains of at most 64 + K / 32 additions, two roundings for each (a matrix
    instruction may round inside), plus the scale's: relative to the sum of magnitudes.  Swish: exp2, reciprocal and
    four products, and the exponent's rounding, which counts |y| times; its slope is at most 1.1.  bf16: half a step."""
    want = x @ w.T
    size = np.abs(x) @ np.abs(w).T
    bound = 2 * EPS32 * (66 + x.shape[1] / 32) * size
    if epilogue:
        with np.errstate(over="ignore"):
            y = want / (1 + np.exp(-want))
        bound = 1.1 * bound + EPS32 * (10 + 2 * np.abs(want)) * np.abs(y)
        want = y
    if y_bf16:
        bound = bound + 2.0 ** -8 * (np.abs(want) + bound)
    bad = np.abs(got - want) > bound + 1e-37  # and what underflows
    assert not bad.any(), (np.argwhere(bad)[:5], np.abs(got - want).max(), bound.max())


# M, N, K around the tiles, groups and units, from one value to long rows
SHAPES = [(1, 1, 1), (1, 3, 31), (1, 17, 33), (2, 64, 32), (1, 512, 512), (1, 100, 150), (1, 130, 2049), (1, 64, 16384), (2, 33, 4090),
          (1, 1000, 64), (1, 9, 20000), (3, 16, 128), (4, 15, 127), (5, 48, 129), (8, 130, 512), (15, 31, 100), (16, 512, 512),
          (16, 16, 16384), (17, 65, 257), (24, 300, 1000), (33, 64, 640), (48, 100, 150), (64, 256, 512), (64, 40, 8200), (65, 70, 96),
          (100, 130, 300), (129, 17, 64), (1, 4099, 96), (2, 5000, 40), (64, 1030, 64),
          # long rows in several rounds or slices, and rows of W that end inside a wavefront's share
          (2, 70, 16384), (1, 5, 40000), (2, 9, 33000), (1, 2000, 1000), (2, 700, 8), (1, 70000, 24), (3, 35, 20000), (20, 40, 5000),
          (64, 9000, 200),
          # many columns and several slices: the most LDS
          (64, 8300, 1100), (33, 17000, 700), (4, 9000, 5000), (16, 16500, 1300)]


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("bf16", [False, True])
def test_product(gpu, shape, group, bf16):
    m, n, k = shape
    rng = np.random.default_rng(m * 31 + n * 7 + k)
    codes, scales = ref.quantize_w4(weights(n, k, n + k), group)
    w = ref.dequantize_w4(codes, scales, k, group)
    x = rng.normal(size=(m, k)).astype(np.float32)
    held = ref.bf16(x) if bf16 else x
    x = (ref.from_bf16(held) if bf16 else held).astype(np.float64)
    check(run(held, codes, scales, group, n, k, bf16, bf16, 0), x, w, bf16, 0)


@pytest.mark.parametrize("x_bf16,y_bf16", [(False, True), (True, False), (False, False), (True, True)])
@pytest.mark.parametrize("m", [1, 2, 7, 16, 40, 80])
def test_product_strides_types_and_swish(gpu, m, x_bf16, y_bf16):
    """odd row strides and starts that are aligned to their elements only; both types mixed; swish"""
    n, k, group = 75, 333, 64
    rng = np.random.default_rng(m)
    codes, scales = ref.quantize_w4(weights(n, k, 3), group)
    w = ref.dequantize_w4(codes, scales, k, group)
    x = (rng.normal(size=(m, k)) * 3).astype(np.float32)
    held = ref.bf16(x) if x_bf16 else x
    x = (ref.from_bf16(held) if x_bf16 else held).astype(np.float64)
    got = run(held, codes, scales, group, n, k, x_bf16, y_bf16, 1, ldx=k + 2 + m % 2, ldy=n + 4, shift=1)
    check(got, x, w, y_bf16, 1)


@pytest.mark.parametrize("m", [1, 2, 5, 20])
def test_product_keeps_the_precision_of_fp32(gpu, m):
    """inputs over many powers of two: nothing is rounded to fewer bits on the way"""
    n, k = 40, 700
    rng = np.random.default_rng(m)
    codes, scales = ref.quantize_w4(weights(n, k, 4), 32)
    w = ref.dequantize_w4(codes, scales, k, 32)
    x = (rng.normal(size=(m, k)) * 10.0 ** rng.uniform(-10, 10, (m, k))).astype(np.float32)
    check(run(x, codes, scales, 32, n, k, False, False, 0), x.astype(np.float64), w, False, 0)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("m", [1, 2, 3, 20])
def test_product_of_subnormal_inputs(gpu, m, bf16):
    """X down to the smallest fp32 numbers against weights that are as large: no part of an input is taken for zero.  What
    is below 2^-126 is exact as an input and in products, so the bound is check's, as for other inputs."""
    n, k = 20, 200
    rng = np.random.default_rng(m)
    codes, scales = ref.quantize_w4((weights(n, k, 4) * np.float32(1e30)).astype(np.float32), 32)
    w = ref.dequantize_w4(codes, scales, k, 32)
    x = (rng.normal(size=(m, k)) * 10.0 ** rng.uniform(-42, -33, (m, k))).astype(np.float32)
    held = ref.bf16(x) if bf16 else x
    got = run(held, codes, scales, 32, n, k, bf16, False, 0)
    check(got, (ref.from_bf16(held) if bf16 else x).astype(np.float64), w, False, 0)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("m", [1, 2, 6, 33])
def test_values_that_are_not_finite(gpu, m, bf16):
    """an infinity or NaN in a row of X reaches that row of Y alone, as the formula has it; a NaN scale its own row of W"""
    n, k, group = 37, 200, 32
    rng = np.random.default_rng(m)
    codes, scales = ref.quantize_w4(weights(n, k, 5), group)
    scales[n - 1, 2] = 0x7FC0
    w = ref.dequantize_w4(codes, scales, k, group)
    x = rng.normal(size=(m, k)).astype(np.float32)
    x[0, 5] = np.inf
    if m > 2:
        x[2, 150] = np.nan
    held = ref.bf16(np.where(np.isfinite(x), x, 0)) if bf16 else x
    if bf16:
        held[~np.isfinite(x)] = 0x7FC0
        held[np.isinf(x)] = 0x7F80
        x = ref.from_bf16(held)
    got = run(held, codes, scales, group, n, k, bf16, False, 0)
    with np.errstate(all="ignore"):
        want = np.stack([[(x[i].astype(np.float64) * w[j]).sum() for j in range(n)] for i in range(m)])
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[np.isinf(want)], want[np.isinf(want)])
    fine = np.isfinite(want)
    with np.errstate(all="ignore"):
        bound = 2 * EPS32 * (66 + k / 32) * (np.abs(x.astype(np.float64)) @ np.abs(w).T)
    assert (np.abs(got - want)[fine] <= bound[fine]).all()


@pytest.mark.parametrize("m", [1, 2, 16, 64])
def test_same_bits_twice(gpu, m):
    rng = np.random.default_rng(1)
    codes, scales = ref.quantize_w4(weights(300, 5000, 6), 64)
    x = rng.normal(size=(m, 5000)).astype(np.float32)
    a, b = (run(x, codes, scales, 64, 300, 5000, False, False, 0) for _ in range(2))
    assert np.array_equal(a, b)


def test_more_rows_than_a_launch_takes(gpu):
    m, n, k = 65535 * 64 + 70, 3, 5
    rng = np.random.default_rng(8)
    codes, scales = ref.quantize_w4(weights(n, k, 9), 32)
    x = rng.normal(size=(m, k)).astype(np.float32)
    check(run(x, codes, scales, 32, n, k, False, False, 0), x.astype(np.float64), ref.dequantize_w4(codes, scales, k, 32), False, 0)


def test_codes_past_four_gib(gpu):
    """rows of W behind 2^32 bytes of codes, and their scales, in each kernel"""
    torch = pytest.importorskip("torch")
    from nerf_amd._lib import lib
    n, k, group = 66000, 131072, 128
    gen = torch.Generator(device="cuda").manual_seed(3)
    codes = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device="cuda", generator=gen)
    scales = torch.randint(0x3C00, 0x4000, (n, k // group), dtype=torch.int16, device="cuda", generator=gen)
    assert codes.numel() > 2 ** 32
    rows = [0, 1000, 65535, 65536, 65999]
    w = ref.dequantize_w4(codes[rows].cpu().numpy(), scales[rows].cpu().numpy().view(np.uint16), k, group)
    for m in (1, 3, 20):
        x = torch.randn(m, k, device="cuda", generator=gen)
        y = torch.empty(m, n, device="cuda")
        size = lib.nerf_gemm_w4_workspace(m, n, k)
        ws = torch.empty(size + 16, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        assert lib.nerf_gemm_w4(x.data_ptr(), 0, k, codes.data_ptr(), scales.data_ptr(), group, y.data_ptr(), 0, n, m, n, k, 0,
                                ws.data_ptr(), size) == 0
        torch.cuda.synchronize()
        check(y[:, rows].cpu().numpy(), x.cpu().numpy().astype(np.float64), w, False, 0)
    del codes, scales, x, y, ws
    torch.cuda.empty_cache()


@pytest.mark.parametrize("m", [1, 24])
def test_graphs_and_streams(gpu, m):
    """quantize, a product (of 24 rows: with parts and their join) and dequantize in one graph on another stream than the
    default, replayed with other weights in place each time, other work in between"""
    import ctypes as C
    torch = pytest.importorskip("torch")
    from nerf_amd._lib import lib
    n, k, group = 300, 2050, 64
    size = lib.nerf_gemm_w4_workspace(m, n, k)
    assert (size > 0) == (m == 24)
    new = lambda shape, t: torch.empty(shape, dtype=t, device="cuda")
    src, x = new((n, k), torch.float32), torch.randn(m, k, device="cuda")

    def buffers():
        return (new((n, lib.nerf_w4_row_bytes(k)), torch.uint8), new((n, -(-k // group)), torch.int16), new((m, n), torch.float32),
                new((n, k), torch.float32), new(size + 16, torch.uint8))

    def calls(codes, scales, y, back, ws):
        return (lib.nerf_quantize_w4(src.data_ptr(), k, n, k, group, codes.data_ptr(), scales.data_ptr()),
                lib.nerf_gemm_w4(x.data_ptr(), 0, k, codes.data_ptr(), scales.data_ptr(), group, y.data_ptr(), 0, n, m, n, k, 0,
                                 ws.data_ptr(), size),
                lib.nerf_dequantize_w4(codes.data_ptr(), scales.data_ptr(), n, k, group, back.data_ptr(), k))

    mine, other = buffers(), buffers()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    src.normal_()
    torch.cuda.synchronize()
    try:
        with torch.cuda.graph(graph, stream=side):
            lib.nerf_set_stream(C.c_void_p(side.cuda_stream))
            assert calls(*mine) == (0, 0, 0)
    finally:
        lib.nerf_set_stream(None)
    for _ in range(3):
        src.normal_()
        for b in mine:
            b.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert calls(*other) == (0, 0, 0)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(mine[:4], other[:4])) and mine[2].abs().max() > 0


def test_trained_with_8_bit_states_and_answered_in_4_bits(gpu):
    """the operators together: gradients of the trainer, their norm, a clipped 8-bit step on its weights, those weights in
    4 bits, and their products with one point and with a few"""
    from conftest import make_scene
    from nerf_amd._lib import lib
    from nerf_amd.api import AdamW, DeviceArray, HostDataset, Trainer, make_camera, trainer_config
    cams, images = make_scene(3, 32, 24)
    dds = HostDataset([make_camera(*c) for c in cams], images).upload()
    tr = Trainer(trainer_config(rays_per_batch=8))
    tr.init_weights(seed=2)
    tensors, shapes = [], []
    for o, (rows, cols) in tr.param_slices():
        size, blocks = rows * cols, lib.nerf_adamw_state_blocks(rows * cols)
        states = {s: DeviceArray.zeros(c, np.uint8) for s, c in (("m", size), ("v", size), ("m_exp", blocks), ("v_exp", blocks))}
        tensors.append(dict(w=tr.params_ptr() + 4 * o, g=tr.grads_ptr() + 4 * o, n=size, **states))
        shapes.append((o, rows, cols))
    plan, norm = AdamW(tensors, state_bits=8), DeviceArray.zeros(1)
    rng = np.random.default_rng(0)
    before = tr.get_params()
    for step in range(1, 3):
        idx = np.stack([rng.integers(0, 3, 8), rng.integers(0, 32, 8), rng.integers(0, 24, 8)], axis=1).astype(np.int32)
        tr.forward_backward(dds, DeviceArray.from_numpy(idx))
        plan.grad_norm(norm, float(tr.N))
        plan.step(step, 1e-3, float(tr.N), norm, 1e-3, seed=3)
    params = tr.get_params()
    assert (params != before).mean() > 0.9
    for o, rows, cols in shapes:
        w = params[o:o + rows * cols].reshape(rows, cols)
        codes, scales = ref.quantize_w4(w, 64)
        d_c, d_s = DeviceArray(codes.shape, np.uint8), DeviceArray(scales.shape, np.uint16)
        assert lib.nerf_quantize_w4(tr.params_ptr() + 4 * o, cols, rows, cols, 64, d_c.ptr, d_s.ptr) == 0
        assert np.array_equal(d_c.numpy(), codes) and np.array_equal(d_s.numpy(), scales)
        for m in (1, 5):
            x = rng.normal(size=(m, cols)).astype(np.float32)
            check(run(x, d_c.numpy(), d_s.numpy(), 64, rows, cols, False, False, 0), x.astype(np.float64),
                  ref.dequantize_w4(codes, scales, cols, 64), False, 0)


def test_a_model_in_4_bits(gpu):
    """the default model's two MLPs in 4 bits, quantized on the device: the run of products that answers a few points,
    against forward_pass_mlp of MLPs that hold the dequantized weights"""
    import ctypes as C
    from nerf_amd._lib import lib
    from nerf_amd.api import DeviceArray, Trainer, device_to_numpy, trainer_config
    rng = np.random.default_rng(3)
    tr = Trainer(trainer_config())
    tr.init_weights(seed=5)
    points = 5
    d_x = DeviceArray.from_numpy(rng.uniform(-1, 1, (points, tr.pe_dim)).astype(np.float32))
    held, mlps = [], []
    for which in (0, 1):
        mlp = tr.mlp(which)
        copy = lib.init_mlp(mlp.input_dim, mlp.hidden_dim, mlp.output_dim, points, None)
        for src, dst, n, k in ((mlp.d_W1, copy.contents.d_W1, mlp.hidden_dim, mlp.input_dim),
                               (mlp.d_W2, copy.contents.d_W2, mlp.output_dim, mlp.hidden_dim)):
            codes, scales = DeviceArray((n, lib.nerf_w4_row_bytes(k)), np.uint8), DeviceArray((n, -(-k // 64)), np.uint16)
            assert lib.nerf_quantize_w4(src, k, n, k, 64, codes.ptr, scales.ptr) == 0
            assert lib.nerf_dequantize_w4(codes.ptr, scales.ptr, n, k, 64, dst, k) == 0
            held.append((codes, scales, n, k))
        mlps.append(copy)
    ws = DeviceArray(max([1] + [lib.nerf_gemm_w4_workspace(points, n, k) for _, _, n, k in held]), np.uint8)
    x = d_x
    for i, (codes, scales, n, k) in enumerate(held):
        y = DeviceArray((points, n))
        assert lib.nerf_gemm_w4(x.ptr, 0, k, codes.ptr, scales.ptr, 64, y.ptr, 0, n, points, n, k, int(i % 2 == 0), ws.ptr, ws.nbytes) == 0
        x = y
    lib.forward_pass_mlp(mlps[0], d_x.ptr)
    lib.forward_pass_mlp(mlps[1], mlps[0].contents.d_layer_output)
    want = device_to_numpy(mlps[1].contents.d_layer_output, (points, 4))
    got = x.numpy()
    # four layers of at most 512 terms: each side within 4 * 512 * EPS32 of the magnitudes, which the layers pass on
    assert np.abs(got - want).max() <= 1e-4 * np.abs(want).max()
    for m in mlps:
        lib.free_mlp(m)
