"""hk_pages_attention and hk_matmul_four at the ends of the ranges that the header states."""
import numpy as np
import pytest

from pages_lib import Pages, filled, within
from test_gpu_four import four, product

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [40, 1000, 6000])
def test_values_whose_sum_is_just_within_float32(n):
    """equal scores: the undivided sum of n values of 3.2e38 / n; a channel past the range is not finite, and no other. Off by a
    rounding of each addition (n at most in all), above and below the division, and its own"""
    model = filled(np.random.default_rng(n), 1, 1, 32, 32, False, [n])
    value = np.float32(3.2e38 / n)
    model.values[:] = value
    model.values[..., 1] = -value
    model.values[..., 2] = np.float32(3e38)
    got = Pages(model).attention(0, np.zeros((1, 64), dtype=np.float32), None, [n], 2)
    keep = np.arange(32) != 2
    want = np.where(np.arange(32) == 1, -1.0, 1.0) * np.float64(value)
    assert (np.abs(got[0, :, keep] - want[keep, None]) <= 2 * (n + 8) * 2.0 ** -24 * np.float64(value)).all()
    assert not np.isfinite(got[0, :, 2]).any()


@pytest.mark.parametrize("length", [40, 1500])
def test_a_half_key_of_minus_infinity_is_nan_or_has_no_weight(length):
    rng = np.random.default_rng(16)
    model = filled(rng, 1, 2, 32, 32, True, [length, length])
    q = np.abs(rng.standard_normal((2, 8 * 32))).astype(np.float32) + np.float32(0.1)
    model.keys[0, model.tables[0, 1], 1, 3, 5] = -np.inf  # position 35 of sequence 0, kv head 1
    got = Pages(model).attention(0, q, None, [length, length], 8)
    model.keys[0, model.tables[0, 1], 1, 3] = -6e4
    want, off = model.attention(0, q, None, [length, length], 8)
    lost = np.isnan(got).all(-1)
    assert not lost[0, :4].any() and not lost[1].any()  # (the other kv head's heads, and the other row)
    assert (np.abs(got - want) <= off)[~lost].all()


@pytest.mark.parametrize("m", [1, 5, 40])
def test_products_of_large_numbers(m):
    """y up to 2e37, of which sixteen times is within float32"""
    rng = np.random.default_rng(m)
    rows, k = 40, 1024
    xq = rng.integers(-127, 128, (m, k)).astype(np.int8)
    w = rng.integers(0, 256, (rows, k // 2)).astype(np.uint8)
    ws, xs = np.full((rows, k // 32), 1e3, dtype=np.float32), np.full((m, k // 32), 1.0, dtype=np.float32)
    largest, _ = product(xq, xs, w, ws, k, 0, 32)
    parts = product(np.abs(xq.astype(np.int64)), xs, w, ws, k, 0, 32)[1].max() * 2.0 ** 24 / (k // 32 + 6)
    xs *= np.float32(2e37 / parts)  # (every partial sum within it)
    want, off = product(xq, xs, w, ws, k, 0, 32)
    got = four(xq, xs, w, ws, rows, k, 0, 32)
    assert np.isfinite(got).all() and (np.abs(got - want) <= off).all() and np.abs(got).max() > 1e36
