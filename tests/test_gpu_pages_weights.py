"""hk_pages_attention where many positions weigh the same: keys that repeat from block to block, whose softmax is the mean of the
values whatever their score is."""
import numpy as np
import pytest

from pages_lib import Model, Pages

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # of a value, a float32 rounding
CHANNELS = 64


def halves(half, kv_heads, n, page=64):
    """one sequence of n positions, all keys 1, values 1 in its first half (channels 0 to 31) and in its second (the others)"""
    slots = -(-n // page)
    model = Model(1, slots, kv_heads, page, CHANNELS, half, 1, slots)
    model.tables[0] = np.random.default_rng(n).permutation(slots)
    model.refs[:] = 1
    model.keys[:] = 1
    for slot, held in enumerate(model.tables[0]):
        first = (slot * page + np.arange(page) < n // 2)[None, :, None]
        model.values[0, held, :, :, :32] = first
        model.values[0, held, :, :, 32:] = ~first
    return model


def queries(scores, rows, group):
    """rows of queries whose heads have the given scores against keys of 1 (all alike in a row)"""
    q = np.repeat(np.asarray(scores, dtype=np.float32) / np.float32(8), CHANNELS).reshape(1, -1)
    return np.ascontiguousarray(np.broadcast_to(q, (rows, q.size)))


def means(got, off):
    """both halves weigh one half, and the same: every position's probability has the same bits, and the accumulators of
    channels 0 to 31 take the additions in the first half that those of 32 to 63 take in the second"""
    np.testing.assert_array_equal(got[..., :32], got[..., 32:])
    assert (np.abs(got - 0.5) <= off).all(), np.abs(got - 0.5).max()


# 32 scores from 3 to 1e5: of about half of them the product with log2(e) lies above its float32, of the others below
SCORES = [float(np.float32(3.3 * 1.395 ** i)) for i in range(32)]


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("rows, n", [(96, 8192), (1, 8192), (300, 4096), (1, 1024), (2, 512)])
def test_keys_that_repeat_weigh_the_same(rows, n, half):
    """in a piece of 64 blocks a wave, and in several; halves that the pieces and their waves take alike. Off the mean by at most
    a rounding of each addition that an accumulator takes, above and below the division: a wave's positions, its products'
    pieces (n / 4 in all at most), the four waves, 16 threads of the join and at most 32 pieces each, the division"""
    model = halves(half, 8, n)
    got = Pages(model).attention(0, queries(SCORES, rows, 4), [0] * rows, [n] * rows, 32)
    means(got, (n / 4 + 4 + 16 + 32 + 1) * U)
    np.testing.assert_array_equal(got, got[:1].repeat(rows, 0))


@pytest.mark.parametrize("half", [False, True])
def test_keys_that_repeat_beside_a_score_that_grows(half):
    """a head whose score rises by more than 2^9 from a wave's block to its next, so that its reference moves every time; the other
    heads' columns of the same products have the same score everywhere. One kv head: the rows are cut into pieces of 9 blocks
    a wave at most (96 rows of 64 units over the 720 or more workgroups that the launch plans), which do not end where the halves
    do. So the halves' sums are not alike to the bit; each is off by at most a rounding of each addition, above and below the
    division: 9 x 32 positions, four waves, 16 of the join, the division"""
    n, rows = 8192, 96
    model = halves(half, 1, n)
    for slot, held in enumerate(model.tables[0]):
        model.keys[0, held, 0, :, 0] = (slot * 64 + np.arange(64)) // 32
    q = queries(SCORES[::4] * 2, rows, 16).reshape(rows, 16, CHANNELS).copy()
    q[:, :, 0] = 0
    q[:, [0, 8]] = 0
    q[:, [0, 8], 0] = 16  # (2 a block in nats, 8 from a wave's to its next: 11.5 in log2)
    others = [h for h in range(16) if h % 8]
    got = Pages(model).attention(0, q.reshape(rows, -1), [0] * rows, [n] * rows, 16)
    off = (9 * 32 + 4 + 16 + 1) * U
    assert (np.abs(got[:, others] - 0.5) <= off).all(), np.abs(got[:, others] - 0.5).max()
    # of the growing heads' positions the last block's weigh alike, one before it by e^-2, and so on
    weight = np.exp(-2.0 * np.arange(n // 32))[::-1].repeat(32)
    want = (weight[n // 2:].sum() / weight.sum())
    assert (np.abs(got[:, [0, 8], 32:] - want) <= 2 * off).all() and (got[:, [0, 8], :32] <= 1e-30).all()


# (float32's whole numbers are two apart from 2^24 on; ordinary scores beside them in the same products)
HUGE = [1e7, -2.3e7, 3e8, 3.3, 1.1e9, -1.1e9, 30.3, 5.3e10, 7.7e20, -100.7, -7.7e30, 377.3] * 2 + [-5.3e10, 2.0 ** 30, 0.0, -2.0 ** 40] * 2


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("rows, n", [(1, 512), (1, 8192), (96, 8192)])
def test_huge_scores_that_repeat_weigh_the_same(rows, n, half):
    got = Pages(halves(half, 8, n)).attention(0, queries(HUGE, rows, 4), [0] * rows, [n] * rows, 32)
    means(got, (n / 4 + 4 + 16 + 32 + 1) * U)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("score", [1e7, 3e8, 1.1e9, 5.3e10, 7.7e20, 7.7e30])
@pytest.mark.parametrize("sign", [1, -1])
def test_one_huge_score_takes_all(score, sign, half):
    """a key of 2 among keys of 1 (of 1 among keys of 2, where the scores are negative): its values. Off by the roundings of its
    probability's halves (2^-23), of their products with the value and their sums (4), of the joins (2) and the division"""
    rng, n = np.random.default_rng(21), 1030
    model = Model(1, 20, 1, 64, CHANNELS, half, 1, 17, rng)
    model.tables[0] = rng.permutation(20)[:17]
    q = queries([sign * score, 0.25 * sign * score], 1, 2)
    for position in (0, 31, 500, 511, 1029):
        model.keys[:] = 1 if sign > 0 else 2
        held = model.tables[0, position // 64]
        model.keys[0, held, 0, position % 64] = 2 if sign > 0 else 1
        want = model.values[0, held, 0, position % 64].astype(np.float64)
        got = Pages(model).attention(0, q, None, [n], 2)
        assert (np.abs(got - want) <= 10 * U * np.abs(want)).all()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("step", [1e7, -1e7, 1e9, -1e9, 1e20])
def test_huge_scores_that_rise_and_fall(step, half):
    """from position to position by more than float32 leaves between them: the first's or the last's values"""
    rng, n = np.random.default_rng(22), 1030
    model = Model(1, 17, 1, 64, CHANNELS, half, 1, 17, rng)
    model.tables[0] = rng.permutation(17)
    model.keys[:] = 0
    for slot, held in enumerate(model.tables[0]):
        model.keys[0, held, 0, :, 3] = slot * 64 + np.arange(64)
    q = np.zeros((1, 2 * CHANNELS), dtype=np.float32)
    q[0, [3, CHANNELS + 3]] = np.float32(8 * step) * np.float32([1, 0.5])
    best = n - 1 if step > 0 else 0
    want = model.values[0, model.tables[0, best // 64], 0, best % 64].astype(np.float64)
    got = Pages(model).attention(0, q, None, [n], 2)
    assert (np.abs(got - want) <= 10 * U * np.abs(want)).all()
