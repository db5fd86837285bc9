"""hk_logprobs where a workgroup reads its part of a row in several batches (of 4096 logits): many rows, unsplit or in a few parts
each, and very long ones."""
import numpy as np
import pytest

from test_gpu_logprobs import agree, expected, run

pytestmark = pytest.mark.gpu

# (rows, logits): 5 and 8 batches unsplit, 6 a part, 8 a part with rows that start at any float
SIZES = [(640, 20011), (1000, 32000), (512, 50257), (300, 128255)]


def some_agree(x, given, top, rows, **how):
    """agree() of the chosen rows, of a call with all of them"""
    logp, h, ids, logps = run(x, given, top, **how)
    wl, wh, wi, wp = expected(x[rows], given[rows], top)
    np.testing.assert_array_equal(ids[rows], wi)
    for got, want in ((logp[rows], wl), (logps[rows], wp)):  # (the bounds that agree() derives)
        infinite = np.isneginf(want)
        np.testing.assert_array_equal(np.isneginf(got), infinite)
        assert (np.abs(got[~infinite] - want[~infinite]) <= 2.0 ** -17 + 2.0 ** -23 * np.abs(want[~infinite])).all()
    assert (np.abs(h[rows] - wh) <= 2.0 ** -12 + 2.0 ** -22 * wh).all()


@pytest.mark.parametrize("m, n", SIZES)
@pytest.mark.parametrize("top, pad", [(0, 0), (5, 1), (32, 3)])
def test_rows_of_several_batches(m, n, top, pad):
    """ordinary rows; rows ascending and descending over their whole length, all equal, of few values, half banned, with all
    but a few banned, with a far logit in the first, a middle and the last batch"""
    rng = np.random.default_rng(n + top)
    x = (rng.standard_normal((m, n)) * 3).astype(np.float32)
    x[1] = np.linspace(-8, 8, n)
    x[2] = np.linspace(8, -8, n)
    x[3] = 1.25
    x[4] = rng.integers(-3, 3, n)
    x[5, rng.random(n) < 0.5] = -np.inf
    x[6] = -np.inf
    x[6, [n // 3, n - 2, n - 1]] = [1.0, 3.0, 2.0]
    for i, at in enumerate((17, n // 2, n - 1)):
        x[7 + i, at] = 60.0
    x[10] = np.sort(x[10])
    x[11] = np.sort(x[11])[::-1]
    x[12, :n // 2] = -np.inf
    x[13] = np.floor(np.linspace(0, 40, n))  # (ties by the hundred, each group above all before it)
    given = rng.integers(0, n, (m, 2))
    some_agree(x, given, top, np.concatenate([np.arange(20), rng.integers(20, m, 15)]), stride=n + pad)


@pytest.mark.parametrize("m, n", SIZES)
@pytest.mark.parametrize("size", [1.04e6, 1.05e6, 1e30, 3.4028234e38])
def test_rows_that_grow_past_the_first_form_on_the_way(m, n, size):
    """a thread's sums change to the form for logits past 2^20 in a late batch, with sums of earlier ones in hand; rows down
    there from the start; rows of the type's lowest value"""
    rng = np.random.default_rng(m)
    x = (rng.standard_normal((m, n)) * 2).astype(np.float32)
    for i, at in enumerate((3, n // 2, n - 1)):
        x[i, at] = size
    x[3, n - 5000:] += np.float32(size)
    x[4] -= np.float32(size)
    x[5, :n - 3] = -np.float32(size)
    x[6] = -np.float32(size)
    x[7, n // 2:] = -np.float32(size)
    given = rng.integers(0, n, (m, 2))
    given[:3, 0] = [3, n // 2, n - 1]
    some_agree(x, given, 9, np.arange(24))


@pytest.mark.parametrize("m, n", SIZES)
def test_rows_without_probabilities_among_many(m, n):
    rng = np.random.default_rng(n)
    x = (rng.standard_normal((m, n))).astype(np.float32)
    given = rng.integers(0, n, (m, 1))
    clean = run(x, given, 3)
    for i, at in enumerate((0, n // 2, n - 1)):
        x[1 + i, at], x[5 + i, at] = np.nan, np.inf
    x[9] = -np.inf
    dirty, bad = run(x, given, 3), [1, 2, 3, 5, 6, 7, 9]
    others = np.setdiff1d(np.arange(m), bad)
    for got, want in zip(dirty, clean):
        np.testing.assert_array_equal(got[others], want[others])
    for got in (dirty[0], dirty[1], dirty[3]):
        assert np.isnan(got[bad]).all()
    assert (dirty[2][bad] == -1).all()


@pytest.mark.parametrize("n, top", [(9_000_001, 20), (33_000_003, 32)])
def test_a_very_long_row(n, top):
    """one row of two and of seven batches a part"""
    rng = np.random.default_rng(n)
    x = (rng.standard_normal((1, n)) * 3).astype(np.float32)
    agree(x, rng.integers(0, n, (1, 3)), top)
    x[0] = np.sort(x[0])
    agree(x, rng.integers(0, n, (1, 3)), top)
