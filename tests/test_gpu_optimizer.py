"""GPU: AdamW over many tensors (32- and 8-bit states) and the global gradient norm, against the formula in 64 bits,
against numpy's float32 in the same order of operations (bit for bit where a code hangs on it), and the fp32 step
against nerf_trainer_update's bits."""
import ctypes as C

import numpy as np
import pytest

import lowbit_ref as ref

pytestmark = pytest.mark.gpu

EPS32 = 2.0 ** -24  # half a step of fp32, relative
SIZES = {
    "one element": [1],
    "around a block": [255, 256, 257, 3],
    "around a chunk": [1023, 1024, 1025, 4095, 4097],
    "none among them": [0, 5, 0, 700, 0],
    "seventy": [1 + (k * 37) % 900 for k in range(70)],
    "over a million": [1 << 20, 5000, 333, 4096],
}
GUARD = 64


class Arena:
    """host arrays packed back to back in device memory, `shift` elements behind an aligned start, with guard
    elements on both sides that a step must leave alone"""

    def __init__(self, parts, dtype, shift=0):
        from nerf_amd.api import DeviceArray
        self.parts = [np.asarray(p, dtype) for p in parts]
        self.item = np.dtype(dtype).itemsize
        self.start = GUARD + shift
        self.total = sum(p.size for p in self.parts)
        self.pattern = np.frombuffer(b"\x5a" * (self.item * (self.start + self.total + GUARD)), dtype).copy()
        flat = self.pattern.copy()
        if self.total:
            flat[self.start:self.start + self.total] = np.concatenate(self.parts)
        self.dev = DeviceArray.from_numpy(flat)
        at = self.start
        self.ptrs = []
        for p in self.parts:
            self.ptrs.append(self.dev.ptr + at * self.item)
            at += p.size

    def read(self):
        flat = self.dev.numpy()
        a, b = self.start, self.start + self.total
        as_bytes = lambda x: np.ascontiguousarray(x).view(np.uint8)  # noqa: E731
        assert (as_bytes(flat[:a]) == 0x5A).all() and (as_bytes(flat[b:]) == 0x5A).all(), "guard elements were written"
        out, at = [], a
        for p in self.parts:
            out.append(flat[at:at + p.size])
            at += p.size
        return out


class Case:
    def __init__(self, sizes, bits, seed, grad_bf16=False, copy=False, shift=0, scale=1.0, per_tensor=False, gradient=None):
        from nerf_amd.api import AdamW
        rng = np.random.default_rng(seed)
        self.sizes, self.bits = sizes, bits
        self.w = [rng.normal(0, 0.1, n).astype(np.float32) for n in sizes]
        g = [(rng.normal(size=n) * 10.0 ** rng.uniform(-5, 0, n) * scale).astype(np.float32) for n in sizes]
        if gradient:
            gradient(g)
        self.g_bits = [ref.bf16(x) for x in g] if grad_bf16 else None
        self.g = [ref.from_bf16(b) for b in self.g_bits] if grad_bf16 else g
        m = [(0.3 * rng.normal(size=n) * 10.0 ** rng.uniform(-5, 0, n)).astype(np.float32) for n in sizes]
        r = [(10.0 ** rng.uniform(-4, 0, n)).astype(np.float32) for n in sizes]
        self.lr_scale = [0.5 + k % 3 for k in range(len(sizes))] if per_tensor else [1.0] * len(sizes)
        self.decay = [0.01 * (k % 4) for k in range(len(sizes))] if per_tensor else [0.01] * len(sizes)
        self.aw = Arena(self.w, np.float32, shift)
        self.ag = Arena(self.g_bits if grad_bf16 else self.g, np.uint16 if grad_bf16 else np.float32, shift)
        self.a16 = Arena([np.zeros(n) for n in sizes], np.uint16, shift) if copy else None
        if bits == 32:
            self.m, self.v = m, [x * x for x in r]
            self.am, self.av = Arena(self.m, np.float32, shift), Arena(self.v, np.float32, shift)
        else:
            half = 1 << 15
            em, er = [ref.encode_m(x, half) if x.size else (x, x) for x in m], [ref.encode_r(x, half) if x.size else (x, x) for x in r]
            self.m = [ref.decode_m(np.asarray(c, np.int64), e).astype(np.float32) if n else np.zeros(0) for (c, e), n in zip(em, sizes)]
            self.v = [ref.decode(c, 4, e).astype(np.float32) if n else np.zeros(0) for (c, e), n in zip(er, sizes)]  # roots
            self.am, self.av = Arena([c for c, _ in em], np.uint8, shift), Arena([c for c, _ in er], np.uint8, shift)
            self.ame, self.ave = Arena([e for _, e in em], np.uint8, shift), Arena([e for _, e in er], np.uint8, shift)
        tensors = []
        for k, n in enumerate(sizes):
            t = dict(g=self.ag.ptrs[k], n=n, g_bf16=grad_bf16, lr_scale=self.lr_scale[k], weight_decay=self.decay[k],
                     w=self.aw.ptrs[k], m=self.am.ptrs[k], v=self.av.ptrs[k])
            if copy:
                t["w_bf16"] = self.a16.ptrs[k]
            if bits == 8:
                t.update(m_exp=self.ame.ptrs[k], v_exp=self.ave.ptrs[k])
            tensors.append(t)
        self.plan = AdamW(tensors, state_bits=bits)

    def reference(self, k, step, lr, div, factor, dtype):
        return ref.adamw_step(self.w[k], self.g[k], self.m[k], self.v[k], step, np.float32(lr) * np.float32(self.lr_scale[k]), div,
                              factor, decay=self.decay[k], root=self.bits == 8, dtype=dtype)


def check_weights(case, got, step, lr, div, factor):
    """w = w0 (1 - lr wd) - alpha m / (r + eps).  Roundings of half a step each, first order: the first term has three
    (1 - lr wd, its product, the difference); m' has up to six behind its terms (quotient, factor, two products, sum,
    and the factor's own division), r' about four (half of those under the root, the root, the sum), alpha four and
    what 1 - beta^step loses: beta^step is off by one step (2 EPS32) of a number below 1.  lr times lr_scale: one."""
    for k, n in enumerate(case.sizes):
        w, m, v, r = case.reference(k, step, lr, div, factor, np.float64)
        b1, b2 = float(np.float32(0.9)), float(np.float32(0.999))
        in_m = 6 * EPS32 * (np.abs(b1 * case.m[k]) + np.abs(m - b1 * case.m[k]))
        alpha = lr * case.lr_scale[k] * np.sqrt(1 - b2 ** step) / (1 - b1 ** step)
        in_alpha = 8 * EPS32 + 2 * EPS32 / (1 - b1 ** step) + EPS32 / (1 - b2 ** step)
        bound = 4 * EPS32 * np.abs(case.w[k]) + alpha / (r + 1e-8) * (in_m + np.abs(m) * (in_alpha + 6 * EPS32)) + EPS32 * np.abs(w)
        assert (np.abs(got[k] - w) <= bound).all(), (k, n, np.max(np.abs(got[k] - w) / bound))


@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("kind", ["f32", "bf16 gradients and copy, unaligned", "per tensor, divisor 3000, clipped"])
def test_step_32(gpu, sizes, kind):
    sizes = SIZES[sizes]
    mixed, clipped = kind.startswith("bf16"), kind.endswith("clipped")
    case = Case(sizes, 32, 1, grad_bf16=mixed, copy=mixed, shift=1 if mixed else 0, scale=3000.0 if clipped else 1.0,
                per_tensor=clipped)
    step, lr, div, factor, norm = 3, 1e-3, 3000.0 if clipped else 1.0, 1.0, None
    if clipped:
        from nerf_amd.api import DeviceArray
        norm = DeviceArray.from_numpy(np.array([8.0], np.float32))
        factor = 0.3125
    case.plan.step(step, lr, div, norm, 2.5 if clipped else 0.0)
    got = case.aw.read()
    check_weights(case, got, step, lr, div, factor)
    for k, (m, v) in enumerate(zip(case.am.read(), case.av.read())):
        _, m32, v32, _ = case.reference(k, step, lr, div, factor, np.float32)
        assert np.array_equal(m, m32) and np.array_equal(v, v32)  # the stated order of fp32 operations
        _, m64, v64, _ = case.reference(k, step, lr, div, factor, np.float64)
        assert (np.abs(v - v64) <= 8 * EPS32 * v64).all()
        assert (np.abs(m - m64) <= 6 * EPS32 * (np.abs(case.m[k]) + np.abs(m64))).all()
    if mixed:
        assert all(np.array_equal(b, ref.bf16(w)) for b, w in zip(case.a16.read(), got))
    assert all(np.array_equal(a, b) for a, b in zip(case.ag.read(), case.g_bits or case.g))


@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("kind", ["nearest", "stochastic", "bf16 gradients and copy, unaligned", "per tensor, divisor 3000, clipped"])
def test_step_8(gpu, sizes, kind):
    sizes = SIZES[sizes]
    mixed, clipped, seed = kind.startswith("bf16"), kind.endswith("clipped"), 0 if kind == "nearest" else 123456789012345
    case = Case(sizes, 8, 2, grad_bf16=mixed, copy=mixed, shift=3 if mixed else 0, scale=3000.0 if clipped else 1.0, per_tensor=clipped)
    step, lr, div, factor, norm = 40, 1e-3, 3000.0 if clipped else 1.0, 1.0, None
    if clipped:
        from nerf_amd.api import DeviceArray
        norm = DeviceArray.from_numpy(np.array([8.0], np.float32))
        factor = 0.3125
    case.plan.step(step, lr, div, norm, 2.5 if clipped else 0.0, seed)
    got = case.aw.read()
    check_weights(case, got, step, lr, div, factor)
    held = list(zip(case.am.read(), case.ame.read(), case.av.read(), case.ave.read()))
    for k, (m, me, v, ve) in enumerate(held):
        if not sizes[k]:
            continue
        _, m32, _, r32 = case.reference(k, step, lr, div, factor, np.float32)
        share_m, share_r = ref.noise(sizes[k], seed, step, k)
        want_m, want_me = ref.encode_m(m32, share_m)
        want_r, want_re = ref.encode_r(r32, share_r)
        assert np.array_equal(me, want_me) and np.array_equal(ve, want_re), k
        assert np.array_equal(m, want_m) and np.array_equal(v, want_r), k
    if mixed:
        assert all(np.array_equal(b, ref.bf16(w)) for b, w in zip(case.a16.read(), got))
    # the values the codes stand for, back to back
    total = sum(sizes)
    out_m, out_r = Arena([np.zeros(total)], np.uint16, 1), Arena([np.zeros(total)], np.uint16, 1)
    case.plan.read_states(out_m.ptrs[0], out_r.ptrs[0])
    want = np.concatenate([ref.decode_m(m.astype(np.int64), me) for m, me, _, _ in held if m.size])
    assert np.array_equal(ref.from_bf16(out_m.read()[0]).astype(np.float64), want)
    want = np.concatenate([ref.decode(v, 4, ve) for _, _, v, ve in held if v.size])
    assert np.array_equal(ref.from_bf16(out_r.read()[0]).astype(np.float64), want)


def test_first_step_from_zeroed_states(gpu):
    """the start: codes and exponents all zero.  m / (r + eps) is then about sign(g), however small g is"""
    case = Case([1000], 8, 5)
    zero = np.zeros(1000, np.uint8)
    for a, n in ((case.am, 1000), (case.av, 1000), (case.ame, 4), (case.ave, 4)):
        flat = a.pattern.copy()
        flat[a.start:a.start + n] = zero[:n]
        a.dev.upload(flat)
    case.m, case.v = [np.zeros(1000, np.float32)], [np.zeros(1000, np.float32)]
    case.plan.step(1, 1e-3)
    check_weights(case, case.aw.read(), 1, 1e-3, 1.0, 1.0)
    _, m32, _, r32 = case.reference(0, 1, 1e-3, 1.0, 1.0, np.float32)
    half = 1 << 15
    assert np.array_equal(case.am.read()[0], ref.encode_m(m32, half)[0]) and np.array_equal(case.av.read()[0], ref.encode_r(r32, half)[0])
    assert (case.av.read()[0] > 0).all()


def extremes(g):
    g[0][:] = 0.0
    g[0][256:512] = 1e-30          # below what the lowest exponent holds
    g[0][512] = 3e38               # its square is not finite
    g[0][600] = 1e-3               # beside it
    g[0][768:1024] = 1e18
    g[0][1024] = np.nan
    g[0][1025] = np.inf
    g[0][1026] = -np.inf


@pytest.mark.parametrize("seed", [0, 7])
@pytest.mark.parametrize("bits", [32, 8])
def test_extreme_gradients(gpu, bits, seed):
    """zero, tiny, huge and not finite gradients: w follows the formula; a state that is not finite is held as zero
    in 8 bits, and its neighbours are what they would be without it"""
    case = Case([1300], bits, 3, gradient=extremes)
    case.plan.step(2, 1e-2, 1.0, None, 0.0, seed)
    w, m, v, r = case.reference(0, 2, 1e-2, 1.0, 1.0, np.float32)
    got = case.aw.read()[0]
    assert np.array_equal(np.isnan(got), np.isnan(w))
    fine = np.isfinite(w)
    # the host's and numpy's powf may differ by a step each in alpha
    assert (np.abs(got - w)[fine] <= 1e-4 * np.abs(w - case.w[0])[fine] + 2 * EPS32 * np.abs(w[fine])).all()
    if bits == 32:
        assert np.array_equal(case.am.read()[0], m, equal_nan=True) and np.array_equal(case.av.read()[0], v, equal_nan=True)
        return
    share_m, share_r = ref.noise(1300, seed, 2, 0)
    for got, want in (((case.am.read()[0], case.ame.read()[0]), ref.encode_m(np.where(np.isfinite(m), m, 0), share_m)),
                      ((case.av.read()[0], case.ave.read()[0]), ref.encode_r(np.where(np.isfinite(r), r, 0), share_r))):
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("value", [np.nan, np.inf])
def test_step_with_a_norm_that_is_not_finite_changes_nothing(gpu, bits, value):
    from nerf_amd.api import DeviceArray
    case = Case([700, 3], bits, 4, copy=True)
    before = [a.dev.numpy() for a in (case.aw, case.am, case.av, case.a16)]
    case.plan.step(1, 1e-2, 1.0, DeviceArray.from_numpy(np.array([value], np.float32)), 1.0)
    for a, b in zip((case.aw, case.am, case.av, case.a16), before):
        assert np.array_equal(a.dev.numpy(), b)


def test_norm_below_the_limit_changes_no_bit(gpu):
    from nerf_amd.api import DeviceArray
    one, two = Case([5000], 32, 6), Case([5000], 32, 6)
    one.plan.step(9, 1e-3, 7.0)
    two.plan.step(9, 1e-3, 7.0, DeviceArray.from_numpy(np.array([2.0], np.float32)), 2.0)
    assert np.array_equal(one.aw.read()[0], two.aw.read()[0])


@pytest.mark.parametrize("points", [16 * 128, 3000])
def test_same_bits_as_the_trainers_update(gpu, points):
    """three steps over the trainer's arena as four tensors, against nerf_trainer_update on another trainer"""
    from nerf_amd.api import AdamW, DeviceArray, Trainer, device_to_numpy, trainer_config
    rng = np.random.default_rng(8)
    a, b = Trainer(trainer_config()), Trainer(trainer_config())
    for t in (a, b):
        t.init_weights(seed=3)
    m, v = DeviceArray.zeros(b.n_params), DeviceArray.zeros(b.n_params)
    params, grads = b.params_ptr(), b.grads_ptr()
    plan = AdamW([dict(w=params + 4 * o, g=grads + 4 * o, m=m.ptr + 4 * o, v=v.ptr + 4 * o, n=s[0] * s[1]) for o, s in b.param_slices()])
    for step in range(1, 4):
        g = (rng.normal(size=a.n_params) * 100).astype(np.float32)
        for t in (a, b):
            DeviceArray(a.n_params, np.float32, ptr=t.grads_ptr()).upload(g)
        a.update(5e-4, points)
        plan.step(step, 5e-4, float(points))
    assert np.array_equal(a.get_params(), b.get_params())
    mlp = a.mlp(0)
    n = mlp.input_dim * mlp.hidden_dim
    assert np.array_equal(device_to_numpy(mlp.d_W1_m, n), m.numpy()[:n]) and np.array_equal(device_to_numpy(mlp.d_W1_v, n), v.numpy()[:n])


@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("bf16", [False, True])
def test_norm(gpu, sizes, bf16):
    """sums in 64 bits: what is left is the rounding of the result"""
    from nerf_amd.api import AdamW, DeviceArray
    rng = np.random.default_rng(11)
    parts = [(rng.normal(size=n) * 10.0 ** rng.uniform(-12, 12, n)).astype(np.float32) for n in SIZES[sizes]]
    if bf16:
        parts = [ref.bf16(p) for p in parts]
    arena = Arena(parts, np.uint16 if bf16 else np.float32, 1)
    plan = AdamW([dict(g=p, n=len(x), g_bf16=bf16) for p, x in zip(arena.ptrs, parts)], state_bits=0)
    out = DeviceArray.zeros(3)
    got = []
    for _ in range(3):
        plan.grad_norm(out.ptr + 4, 48.0)
        got.append(out.numpy())
        assert got[-1][0] == 0 and got[-1][2] == 0
    flat = np.concatenate([ref.from_bf16(p) if bf16 else p for p in parts]).astype(np.float64)
    want = np.sqrt((flat ** 2).sum()) / 48.0
    assert abs(got[0][1] - want) <= 1.001 * EPS32 * want and all(np.array_equal(g, got[0]) for g in got)


@pytest.mark.parametrize("value,want", [(0.0, 0.0), (np.inf, np.inf), (np.nan, np.nan), (3e38, None)])
def test_norm_of_extremes(gpu, value, want):
    from nerf_amd.api import AdamW, DeviceArray
    g = np.zeros(5000, np.float32)
    g[4321] = value
    d, out = DeviceArray.from_numpy(g), DeviceArray.zeros(1)
    AdamW([dict(g=d, n=5000)], state_bits=0).grad_norm(out)
    want = np.float32(value) if want is None else want
    assert np.array_equal(out.numpy()[0], want, equal_nan=True) or abs(out.numpy()[0] - want) <= EPS32 * abs(want)
    AdamW([dict(g=0, n=0)], state_bits=0).grad_norm(out)
    assert out.numpy()[0] == 0.0


@pytest.mark.parametrize("bits", [32, 8])
def test_norm_then_clipped_step(gpu, bits):
    """the two together, as a training step uses them"""
    from nerf_amd.api import DeviceArray
    case = Case([30000, 77, 4096], bits, 12, scale=5.0)
    norm = DeviceArray.zeros(1)
    case.plan.grad_norm(norm, 5.0)
    case.plan.step(10, 1e-3, 5.0, norm, 0.5)
    flat = np.concatenate(case.g).astype(np.float64) / 5.0
    length = np.sqrt((flat ** 2).sum())
    assert length > 0.5
    check_weights(case, case.aw.read(), 10, 1e-3, 5.0, 0.5 / length)


def test_step_refusals(gpu):
    from nerf_amd._lib import lib
    case, norms = Case([100], 32, 1), None
    before = case.aw.dev.numpy()
    h = case.plan.handle
    nan = float("nan")
    for args in ((0, 0.1, 1.0, None, 0.0), (1, nan, 1.0, None, 0.0), (1, -0.1, 1.0, None, 0.0), (1, 0.1, 0.0, None, 0.0),
                 (1, 0.1, -2.0, None, 0.0), (1, 0.1, nan, None, 0.0), (1, 0.1, 1.0, case.aw.ptrs[0], 0.0),
                 (1, 0.1, 1.0, case.aw.ptrs[0], nan)):
        assert lib.nerf_adamw_step(h, *args, 0) == 1, args
    assert lib.nerf_adamw_read_states(h, case.aw.ptrs[0], None) == 1  # 32-bit states
    assert lib.nerf_grad_norm(h, 1.0, None) == 1 and lib.nerf_grad_norm(h, 0.0, case.aw.ptrs[0]) == 1
    from nerf_amd.api import AdamW
    norms = AdamW([dict(g=case.ag.ptrs[0], n=100)], state_bits=0)
    assert lib.nerf_adamw_step(norms.handle, 1, 0.1, 1.0, None, 0.0, 0) == 1
    assert np.array_equal(case.aw.dev.numpy(), before)
    host = np.zeros(100, np.float32)
    with pytest.raises(RuntimeError):
        AdamW([dict(g=host.ctypes.data, n=100)], state_bits=0)


def test_graphs_and_streams(gpu):
    """the norm is captured and replayed, on another stream than the default; a step is refused while capturing"""
    torch = pytest.importorskip("torch")
    from nerf_amd._lib import lib
    case = Case([50000, 123], 8, 13)
    other = Case([50000, 123], 8, 13)
    norm = torch.zeros(1, device="cuda")
    want = torch.zeros(1, device="cuda")
    case.plan.grad_norm(want.data_ptr(), 2.0)
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    try:
        with torch.cuda.graph(graph, stream=side):
            lib.nerf_set_stream(C.c_void_p(side.cuda_stream))
            case.plan.grad_norm(norm.data_ptr(), 2.0)
            refused = lib.nerf_adamw_step(case.plan.handle, 1, 1e-3, 1.0, None, 0.0, 0)
        assert refused == 1
        for _ in range(3):
            norm.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert norm.item() == want.item() != 0.0
        case.plan.step(4, 1e-3, 2.0, norm.data_ptr(), 0.25, 5)  # on the side stream
        side.synchronize()
    finally:
        lib.nerf_set_stream(None)
    other.plan.step(4, 1e-3, 2.0, want.data_ptr(), 0.25, 5)
    assert np.array_equal(case.aw.read()[0], other.aw.read()[0]) and np.array_equal(case.am.read()[0], other.am.read()[0])


def test_no_plan_is_made_while_a_stream_is_captured(gpu):
    """refused before anything that would end the capture: the norm captured beside it replays"""
    torch = pytest.importorskip("torch")
    from nerf_amd._lib import lib
    from nerf_amd.api import AdamW
    case, norm, want = Case([5000], 32, 3), torch.zeros(1, device="cuda"), torch.zeros(1, device="cuda")
    case.plan.grad_norm(want.data_ptr())
    torch.cuda.synchronize()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    try:
        with torch.cuda.graph(graph, stream=side, capture_error_mode="relaxed"):
            lib.nerf_set_stream(C.c_void_p(side.cuda_stream))
            with pytest.raises(Exception, match="nerf_adamw_create"):
                AdamW([dict(g=norm.data_ptr(), n=1)], state_bits=0)
            case.plan.grad_norm(norm.data_ptr())
    finally:
        lib.nerf_set_stream(None)
    for _ in range(2):
        norm.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert norm.item() == want.item() != 0.0


def test_more_than_2_to_the_32_elements(gpu):
    """one tensor longer than 32 bits count: equal elements stay equal to the end, and the norm counts them all"""
    torch = pytest.importorskip("torch")
    from nerf_amd._lib import lib
    from nerf_amd.api import AdamW
    n = 2 ** 32 + 1030
    blocks = lib.nerf_adamw_state_blocks(n)
    new = lambda count, t: torch.zeros(count, dtype=t, device="cuda")
    w, g = new(n, torch.float32), torch.full((n,), 0.5, dtype=torch.bfloat16, device="cuda")
    m, v, me, ve = new(n, torch.uint8), new(n, torch.uint8), new(blocks, torch.uint8), new(blocks, torch.uint8)
    norm = new(1, torch.float32)
    torch.cuda.synchronize()
    plan = AdamW([dict(w=w.data_ptr(), g=g.data_ptr(), m=m.data_ptr(), v=v.data_ptr(), m_exp=me.data_ptr(), v_exp=ve.data_ptr(), n=n,
                       g_bf16=True)], state_bits=8)
    plan.grad_norm(norm.data_ptr())
    plan.step(1, 1e-2)
    torch.cuda.synchronize()
    assert norm.item() == np.float32(0.5 * np.sqrt(n))
    # m / (sqrt(v) + eps) times the corrections for the first step is 1 to a few roundings
    assert abs(w[0].item() + 1e-2) <= 1e-2 * 16 * EPS32 + 1e-2 * 1e-8 / 0.5
    for t in (w, m, v, me, ve):
        assert bool((t == t[0]).all()) and t[0].item() != 0
    plan.destroy()
    del w, g, m, v, t
    torch.cuda.empty_cache()


def test_training_step_with_8_bit_states(gpu):
    """forward and backward of the trainer, the norm, and the clipped 8-bit step on the trainer's own arenas: three
    steps, each against the formula on the gradients and states the device held before it"""
    from conftest import make_scene
    from nerf_amd.api import AdamW, DeviceArray, HostDataset, Trainer, make_camera, trainer_config
    cams, images = make_scene(3, 32, 24)
    dds = HostDataset([make_camera(*c) for c in cams], images).upload()
    tr = Trainer(trainer_config(rays_per_batch=8))
    tr.init_weights(seed=2)
    sizes = [s[0] * s[1] for _, s in tr.param_slices()]
    blocks = [-(-n // ref.BLOCK) for n in sizes]
    m, v = DeviceArray.zeros(sum(sizes), np.uint8), DeviceArray.zeros(sum(sizes), np.uint8)
    me, ve = DeviceArray.zeros(sum(blocks), np.uint8), DeviceArray.zeros(sum(blocks), np.uint8)
    tensors, b = [], 0
    for (o, _), n, k in zip(tr.param_slices(), sizes, blocks):
        tensors.append(dict(w=tr.params_ptr() + 4 * o, g=tr.grads_ptr() + 4 * o, m=m.ptr + o, v=v.ptr + o, m_exp=me.ptr + b,
                            v_exp=ve.ptr + b, n=n))
        b += k
    plan, norm = AdamW(tensors, state_bits=8), DeviceArray.zeros(1)
    rng = np.random.default_rng(0)
    for step in range(1, 4):
        idx = np.stack([rng.integers(0, 3, 8), rng.integers(0, 32, 8), rng.integers(0, 24, 8)], axis=1).astype(np.int32)
        tr.forward_backward(dds, DeviceArray.from_numpy(idx))
        w0, (g, _) = tr.get_params(), tr.get_grads()
        m0, v0, me0, ve0 = m.numpy(), v.numpy(), me.numpy(), ve.numpy()
        plan.grad_norm(norm, float(tr.N))
        length = np.sqrt((g.astype(np.float64) ** 2).sum()) / tr.N
        plan.step(step, 1e-3, float(tr.N), norm, float(0.5 * length), seed=17)
        w1, o, b = tr.get_params(), 0, 0
        factor = np.float32(0.5 * length) / norm.numpy()[0]
        for k, n in enumerate(sizes):
            mv = ref.decode_m(m0[o:o + n].astype(np.int64), me0[b:b + blocks[k]]).astype(np.float32)
            rv = ref.decode(v0[o:o + n], 4, ve0[b:b + blocks[k]]).astype(np.float32)
            w, m32, _, r32 = ref.adamw_step(w0[o:o + n], g[o:o + n], mv, rv, step, 1e-3, tr.N, factor, root=True, dtype=np.float32)
            share_m, share_r = ref.noise(n, 17, step, k)
            assert np.array_equal(m.numpy()[o:o + n], ref.encode_m(m32, share_m)[0])
            assert np.array_equal(v.numpy()[o:o + n], ref.encode_r(r32, share_r)[0])
            assert np.abs(w1[o:o + n] - w).max() <= 1e-4 * np.abs(w - w0[o:o + n]).max() + 4 * EPS32 * np.abs(w).max()
            o, b = o + n, b + blocks[k]
