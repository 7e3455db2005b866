"""CPU: the plain statement of the 4-bit weights against its definition, and what the entry points refuse (status 1)
before they launch anything; what passes the checks fails with 2 where there is no GPU."""
import numpy as np
import pytest

import lowbit_ref as ref


@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantized_weights_are_the_nearest(group):
    rng = np.random.default_rng(group)
    w = (rng.normal(size=(7, 300)) * 10.0 ** rng.uniform(-30, 30, (7, 1))).astype(np.float32)
    w[3, :group] = 0.0
    codes, scales = ref.quantize_w4(w, group)
    got = ref.dequantize_w4(codes, scales, 300, group)
    scale = np.repeat(ref.from_bf16(scales).astype(np.float64), group, axis=1)[:, :300]
    grid = np.concatenate([-ref.E2M1[::-1], ref.E2M1])
    best = np.abs(grid[None, None, :] * scale[:, :, None] - w.astype(np.float64)[:, :, None]).min(2)
    assert np.array_equal(np.abs(got - w), best)
    assert (np.abs(w) <= 6 * scale).all() and (got[3, :group] == 0).all()


def test_ties_go_to_the_even_code():
    w = np.zeros((1, 32), np.float32)
    w[0, :9] = [6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -2.5]
    codes, scales = ref.quantize_w4(w, 32)
    assert ref.from_bf16(scales)[0, 0] == 1.0
    assert ref.dequantize_w4(codes, scales, 32, 32)[0, :9].tolist() == [6, 0, 1, 1, 2, 2, 4, 4, -2]


GOOD_Q = dict(src=0x1000, ld=100, rows=4, cols=100, group=32, codes=0x2000, scales=0x3000)
BAD_Q = [dict(src=None), dict(codes=None), dict(scales=None), dict(rows=0), dict(cols=-1), dict(ld=99), dict(group=16), dict(group=0),
         dict(src=0x1002), dict(codes=0x2008), dict(scales=0x3001), dict(cols=(1 << 30) + 1, ld=1 << 31)]


@pytest.mark.parametrize("bad", BAD_Q, ids=str)
def test_conversions_refuse(bad):
    from nerf_amd._lib import lib
    q = {**GOOD_Q, **bad}
    assert lib.nerf_quantize_w4(q["src"], q["ld"], q["rows"], q["cols"], q["group"], q["codes"], q["scales"]) == 1
    assert lib.nerf_dequantize_w4(q["codes"], q["scales"], q["rows"], q["cols"], q["group"], q["src"], q["ld"]) == 1


GOOD_P = dict(x=0x1000, xt=0, ldx=100, codes=0x2000, scales=0x3000, group=64, y=0x4000, yt=1, ldy=8, m=3, n=8, k=100, epi=1, ws=0x8000,
              wb=1 << 30)
BAD_P = [dict(x=None), dict(codes=None), dict(scales=None), dict(y=None), dict(m=0), dict(n=0), dict(k=0), dict(ldx=99), dict(ldy=7),
         dict(group=48), dict(xt=2), dict(yt=-1), dict(epi=2), dict(x=0x1002), dict(x=0x1001, xt=1), dict(codes=0x2004),
         dict(scales=0x3001), dict(y=0x4001), dict(y=0x4002, yt=0), dict(ws=0x8004), dict(k=(1 << 30) + 1, ldx=1 << 31), dict(n=(1 << 30) + 1, ldy=1 << 31)]


def _product(lib, p):
    return lib.nerf_gemm_w4(p["x"], p["xt"], p["ldx"], p["codes"], p["scales"], p["group"], p["y"], p["yt"], p["ldy"], p["m"], p["n"],
                            p["k"], p["epi"], p["ws"], p["wb"])


@pytest.mark.parametrize("bad", BAD_P, ids=str)
def test_products_refuse(bad):
    from nerf_amd._lib import lib
    assert _product(lib, {**GOOD_P, **bad}) == 1


def test_products_refuse_a_workspace_that_is_too_small():
    from nerf_amd._lib import lib
    for m, n, k in ((1, 64, 16384), (16, 512, 512), (64, 4096, 8192), (5, 100000, 64)):
        need = lib.nerf_gemm_w4_workspace(m, n, k)
        if need:
            p = {**GOOD_P, "m": m, "n": n, "k": k, "ldx": k, "ldy": n}
            assert _product(lib, {**p, "wb": need - 1}) == 1 and _product(lib, {**p, "ws": None}) == 1
    assert [lib.nerf_w4_row_bytes(k) for k in (0, 1, 32, 33, 150)] == [0, 16, 16, 32, 80]
