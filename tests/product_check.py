"""A check of products that a NaN fails, beside test_gpu_w4.check, whose comparison a NaN passes."""
import numpy as np

import test_gpu_w4 as products

compare = products.check  # the same bound


def check(got, x, w, y_bf16, epilogue):
    """for finite inputs with finite results: every value is a number, and within products.check's bound"""
    assert np.isfinite(got).all(), (np.argwhere(~np.isfinite(got))[:5], got.shape)
    compare(got, x, w, y_bf16, epilogue)
