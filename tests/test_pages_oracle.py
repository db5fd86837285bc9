"""The oracles of long rows see what they are there for: mistakes planted in a second one, on the CPU."""
import numpy as np
import pytest

from pages_exact import close, means, whole
from pages_lib import filled


def without(n, lost):
    """the positions of a row of n but for the lost ones"""
    keep = np.ones(n, dtype=bool)
    keep[lost] = False
    return np.flatnonzero(keep)


@pytest.mark.parametrize("n", [1030, 9000, 33000, 131077])
def test_a_position_that_is_lost_or_doubled_shows_in_the_mean(n):
    model = whole(np.random.default_rng(n), 1, 1, 64, 16, True, [n])
    want = means(model, 0, None, [n], 1)[0, 0]
    _, v = model.rows(0, 0, n)
    v = v[:, 0]
    lists = [without(n, at) for at in (0, 31, 32, 127, 128, n // 2, n - 1)]
    lists += [without(n, np.arange(at, at + 32)) for at in (0, 256, (n // 2) & ~31)] + [np.r_[:n, n - 1], np.r_[:n, 128], np.r_[1:n + 1] % n]
    for i, held in enumerate(lists):
        got = v[held].sum(0).astype(np.float32) / np.float32(len(held))
        if i == len(lists) - 1:  # (all of them, in another order)
            np.testing.assert_array_equal(got, want)
        else:
            assert (got != want).any(), i


@pytest.mark.parametrize("half, n, adds", [(False, 33000, 120), (True, 20011, 120), (True, 9000, 2400)])
def test_a_lost_block_shows_past_the_bound(n, half, adds):
    rng = np.random.default_rng(8)
    model = filled(rng, 1, 1, 128, 64, half, [n])
    q = rng.standard_normal((1, 4 * 64)).astype(np.float32)
    want, off = close(model, 0, q, None, [n], 4, adds)
    k, v = (x[:, 0] for x in model.rows(0, 0, n))
    for lost in (np.arange(32), np.arange(128, 160), np.arange(n // 2, n // 2 + 32), np.arange(n - 32, n), np.arange(n - 10, n)):
        held, worst = without(n, lost), 0.0
        for h in range(4):
            p = np.exp(k[held] @ q.astype(np.float64).reshape(4, 64)[h] / 8)
            worst = max(worst, (np.abs(p @ v[held] / p.sum() - want[0, h]) / off[0, h]).max())
        assert worst > 1.0, (lost[0], worst)
