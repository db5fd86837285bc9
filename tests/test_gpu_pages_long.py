"""hk_pages_attention over long rows, each position of which counts: the mean of whole numbers to the bit, and any queries within a
bound of the outputs' size."""
import numpy as np
import pytest

from pages_exact import close, means, whole
from pages_lib import Pages, filled

pytestmark = pytest.mark.gpu


def equal(model, seqs, lengths, nh, longest=None):
    q = np.zeros((len(lengths), nh * model.hs), dtype=np.float32)
    got = Pages(model).attention(0, q, seqs, lengths, nh, longest=longest)
    np.testing.assert_array_equal(got, means(model, 0, seqs, lengths, nh))


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("nkv, hs, page, lengths", [(1, 64, 128, [20011, 9, 33000]), (1, 64, 64, [131077]), (2, 128, 32, [131077 // 4, 1]),
                                                     (8, 64, 64, [8205, 8191, 640, 641, 1025]), (1, 48, 256, [70001, 128])])
def test_every_position_of_long_rows_counts_once(nkv, hs, page, lengths, half):
    model = whole(np.random.default_rng(sum(lengths)), 1, nkv, page, hs, half, lengths)
    equal(model, None, lengths, 4 * nkv)
    equal(model, list(range(len(lengths))), lengths, nkv, longest=model.slots * page)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("hs", [16, 32, 48, 64, 96, 128, 256])
def test_every_position_counts_at_every_head_size(hs, half):
    lengths = [5001, 640, 641, 129, 2, 0]
    model = whole(np.random.default_rng(hs), 1, 2, 64, hs, half, lengths)
    equal(model, None, lengths, 6)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("rows, nkv, hs, held, longest", [
    (300, 64, 16, 9000, 9000),    # a row one piece, whose waves look up pages a second time
    (96, 8, 64, 8205, 8205),      # planned, a row one piece
    (256, 2, 32, 3000, 3000), (257, 2, 32, 3000, 3000), (700, 2, 32, 3000, 3000), (40, 1, 128, 20000, 20480)])
def test_every_position_counts_in_rows_of_one_sequence(rows, nkv, hs, held, longest, half):
    rng = np.random.default_rng(rows)
    model = whole(rng, 1, nkv, 32, hs, half, [held])
    if longest > model.slots * 32:
        longest = model.slots * 32
    near = [held, held - 1, held // 2, 8193 % held + 1, 8192 % held, 1, 0]
    lengths = near + rng.integers(0, min(held, 2000), rows - len(near)).tolist()
    if rows < 100:
        lengths = near + rng.integers(held // 2, held, rows - len(near)).tolist()
    equal(model, [0] * rows, lengths, nkv, longest=longest)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("lengths, rows, adds", [
    # pieces of two units (64 positions a wave), their join (at most 129 by 16 threads), the waves and threads
    ([20011, 9, 33000], 3, 64 + 9 + 16 + 4 + 1),
    # one piece: a quarter of the row a wave
    ([8205], 96 * 8, 8205 // 4 + 32 + 16 + 4 + 1)])
def test_long_rows_within_a_bound_of_their_size(lengths, rows, adds, half):
    rng = np.random.default_rng(8)
    if rows == 3:
        model, seqs, lens, nh = filled(rng, 1, 1, 128, 64, half, lengths), None, lengths, 4
    else:
        model, seqs, lens, nh = filled(rng, 1, 8, 64, 64, half, lengths), [0] * 96, lengths * 96, 8
    q = rng.standard_normal((len(lens), nh * 64)).astype(np.float32)
    got = Pages(model).attention(0, q, seqs, lens, nh)
    some = range(len(lens)) if rows == 3 else [0, 40, 95]
    want, off = close(model, 0, q[list(some)], seqs and [0] * 3, [lens[i] for i in some], nh, adds)
    assert (np.abs(got[list(some)] - want) <= off).all(), (np.abs(got[list(some)] - want) / off).max()
