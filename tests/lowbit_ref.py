"""Plain statements of the optimizer step over many tensors and of the two low-bit formats, in numpy.

adamw_step works in float64 or, with the same order of operations as the library states, in float32."""
import numpy as np

BLOCK = 256
E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
M_BITS, R_BITS = 3, 4  # mantissa bits of the codes of m and of sqrt(v)


def bf16(x):
    """float32 -> bf16 bit patterns, to nearest with ties to even (finite values)"""
    b = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((b + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)


def from_bf16(b):
    return (np.asarray(b, np.uint16).astype(np.uint32) << 16).view(np.float32)


# ---- 8-bit states ---------------------------------------------------------------------------------------

def _mix(x):
    x = np.asarray(x, np.uint64) & 0xFFFFFFFF
    x ^= x >> np.uint64(16)
    x = (x * np.uint64(0x7FEB352D)) & np.uint64(0xFFFFFFFF)
    x ^= x >> np.uint64(15)
    x = (x * np.uint64(0x846CA68B)) & np.uint64(0xFFFFFFFF)
    return x ^ (x >> np.uint64(16))


def noise(n, seed, step, tensor):
    """(share of a step added to |m|, to sqrt(v)) before the fraction is dropped, in units of 2^-16 steps"""
    if seed == 0:
        half = np.full(n, 1 << 15, np.int64)
        return half, half
    u = (1 << 64) - 1
    z = (seed + step * 0x9E3779B97F4A7C15) & u
    z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & u
    z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & u
    z ^= z >> 31
    key = (z ^ (z >> 32)) & 0xFFFFFFFF
    i = np.arange(n)
    of_tensor = int(_mix(key + tensor * 0x9E3779B9))
    of_block = _mix((of_tensor + (i // BLOCK) * 0x85EBCA6B) & 0xFFFFFFFF)
    h = _mix(of_block ^ (i % BLOCK).astype(np.uint64)).astype(np.int64)
    return h & 0xFFFF, h >> 16


def exponents(x, bits):
    """a block's biased exponent: the smallest whose largest code is at least the largest value, in 16..254"""
    x = np.where(np.isfinite(x), np.abs(x), 0).astype(np.float64)
    top = np.array([x[b:b + BLOCK].max() for b in range(0, len(x), BLOCK)])
    e = np.frexp(top)[1] - 1
    e = e + (top > (2 - 2.0 ** -bits) * 2.0 ** e.astype(np.float64))
    return np.where(top > 0, np.clip(e + 127, 16, 254), 16).astype(np.uint8)


def encode(x, bits, exps, share):
    """codes of x >= 0 (float32 values); `share` in 2^-16 steps"""
    e = np.repeat(exps.astype(np.int64) - 127, BLOCK)[: len(x)]
    x = np.where(np.isfinite(x), x, 0).astype(np.float64)
    own = np.where(x > 0, np.maximum(np.frexp(x)[1] - 1, e - 14), e - 14)
    n = np.floor(x * 2.0 ** (bits - own) + share / 65536.0).astype(np.int64)  # of steps in the value's own binade
    code = n + ((own - (e - 14)) << bits)
    return np.minimum(code, (16 << bits) - 1)


def decode(code, bits, exps):
    e = np.repeat(exps.astype(np.int64) - 127, BLOCK)[: len(code)].astype(np.float64)
    code = np.asarray(code, np.int64)
    field, fraction = code >> bits, (code & ((1 << bits) - 1)) / 2.0 ** bits
    return np.where(field > 0, (1 + fraction) * 2.0 ** (field - 15.0), fraction * 2.0 ** -14) * 2.0 ** e


def decode_m(codes, exps):
    v = decode(codes & 127, M_BITS, exps)
    return np.where(codes > 127, -v, v)


def encode_m(m, share):
    exps = exponents(m, M_BITS)
    c = encode(np.abs(m), M_BITS, exps, share)
    return np.where((m < 0) & (c > 0), c + 128, c).astype(np.uint8), exps


def encode_r(r, share):
    exps = exponents(r, R_BITS)
    c = encode(r, R_BITS, exps, share)
    return np.where((c == 0) & (r > 0) & np.isfinite(r), 1, c).astype(np.uint8), exps


# ---- the step -------------------------------------------------------------------------------------------

def adamw_step(w, g, m, r_or_v, step, lr, div, factor=1.0, beta1=0.9, beta2=0.999, eps=1e-8, decay=0.01, root=False,
               dtype=np.float64):
    """(w, m, v, sqrt(v)) after one step; root: the second moment comes as its square root"""
    f = dtype
    b1, b2 = f(np.float32(beta1)), f(np.float32(beta2))
    lr, eps, decay = f(np.float32(lr)), f(np.float32(eps)), f(np.float32(decay))
    w, m = w.astype(f), m.astype(f)
    v = r_or_v.astype(f)
    if root:
        v = v * v
    with np.errstate(all="ignore"):
        gi = g.astype(f) / f(np.float32(div)) * f(factor)
        m = b1 * m + (f(1) - b1) * gi
        v = b2 * v + ((f(1) - b2) * gi) * gi
        alpha = lr * np.sqrt(f(1) - b2 ** f(step)) / (f(1) - b1 ** f(step))
        r = np.sqrt(v)
        w = w * (f(1) - lr * decay) - alpha * m / (r + eps)
    return w, m, v, r


# ---- 4-bit weights --------------------------------------------------------------------------------------

def w4_row_bytes(k):
    return -(-k // 32) * 16


def quantize_w4(w, group):
    """(codes [n][row bytes], scales as bf16 bits [n][groups]) of a float32 [n][k] matrix"""
    n, k = w.shape
    groups = -(-k // group)
    x = np.zeros((n, groups * group))
    x[:, :k] = w
    x = x.reshape(n, groups, group)
    top = np.abs(x).max(2)
    bad = ~np.isfinite(x).all(2)
    bits = np.zeros(top.shape, np.uint32)
    with np.errstate(all="ignore"):
        bits = (np.where(bad, 0, top) / 6).astype(np.float32).view(np.uint32) >> 16
        value = lambda b: (b << 16).view(np.float32).astype(np.float64)  # noqa: E731
        for _ in range(2):
            bits = np.where((bits > 0) & (6 * value(np.maximum(bits, 1) - 1) >= np.where(bad, 0, top)), bits - 1, bits)
        for _ in range(2):
            bits = np.where(6 * value(bits) < np.where(bad, 0, top), bits + 1, bits)
    scale = value(bits)[:, :, None]
    a = np.abs(np.where(bad[:, :, None], 0, x))
    edges = [(0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)]
    code = sum(((a >= t * scale) if at else (a > t * scale)).astype(np.int64) for t, at in edges)
    code = np.where(scale > 0, code, 0)
    code = np.where((x < 0) & (code > 0), code + 8, code).reshape(n, -1)
    bits = np.where(bad, 0x7FC0, bits).astype(np.uint16)
    full = np.zeros((n, 2 * w4_row_bytes(k)), np.int64)
    full[:, :k] = code[:, :k]
    return (full[:, 0::2] | (full[:, 1::2] << 4)).astype(np.uint8), bits


def dequantize_w4(codes, scales, k, group):
    n = codes.shape[0]
    both = np.stack([codes & 15, codes >> 4], axis=2).reshape(n, -1)[:, :k]
    value = np.where(both > 7, -1.0, 1.0) * E2M1[both & 7]
    return value * np.repeat(from_bf16(scales).astype(np.float64), group, axis=1)[:, :k]
