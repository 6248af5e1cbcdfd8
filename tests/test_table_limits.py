"""The operators over whole tables at the limits of their number ranges and lengths: tables that callers make themselves, products near
the end of the f32 range, tables long enough for a sum to forget, tables worked on in pieces."""
import numpy as np
import pytest

from tests import table_ref as R
from tests.test_quantized import METRICS, _check_knn, _gpu_table


# ---- scores of a large batch ---------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("metric", METRICS)
@pytest.mark.parametrize("B", [5, 40, 300])
def test_groups_of_zeros_with_large_scales(gpu_lib, metric, B):
    """a group whose codes are all zero may have any scale, and what stands in the padding does not count: such rows, each the nearest one
    and alone in its tile, are found"""
    n, dim, group = 33000, 72, 32
    rng = np.random.default_rng(B)
    c = rng.integers(-7, 8, (n, 96))
    u = rng.integers(1, 8, 32)
    c[c[:, :32] @ u > 0] *= -1  # all others point away
    c[:, dim:] = rng.integers(-8, 8, (n, 96 - dim))  # the padding
    s = np.exp(rng.uniform(-1, 2, (n, 3)))
    at = np.array([70, 6400, 12801, 20031, 32999])
    # 1e-3 in all, beside a group of zeros with a scale up to the largest bfloat16 numbers
    c[at, :] = 0
    c[at, :32] = u
    s[at, 0] = 1e-3 / np.linalg.norm(u) * (1 + 0.05 * np.arange(5))
    s[at, 1] = [1.0, 1e30, 1.0, 3e38, 1.0]
    s[at, 2] = [1.0, 1.0, 1e30, 3e38, 1e6]
    c[at[2:], dim:] = 7
    c[at[3], dim:] = -8
    scales = R.bf16_bits(s.astype(np.float32))
    codes = R.pack(c)
    x = R.decode(codes, R.bf16_value(scales), dim)
    t = _gpu_table(codes, scales, (x ** 2).sum(1).astype(np.float32), dim)
    q = np.zeros((B, dim), np.float32)
    q[:, :32] = u * np.exp(rng.uniform(-1, 1, (B, 1))) * 1e-3 / np.linalg.norm(u)
    look = np.arange(0, B, max(1, B // 8))
    for k in (1, 5, 20):
        ids, _ = _check_knn(t, q, x, k, metric, only=look)
        assert np.isin(ids[:, :min(k, 5)], at).all()
