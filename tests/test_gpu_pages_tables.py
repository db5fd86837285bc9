"""hk_pages_*: the largest tables, and calls one after the other whose answers a program reads later."""
import numpy as np
import pytest

from gpu_lib import check
from pages_lib import Model, Pages, filled, ints

pytestmark = pytest.mark.gpu


def test_a_fork_of_the_longest_tables_by_a_list_that_is_filled_up():
    """2^25 slots a sequence, and so many entries listed that a workgroup takes one slot at a time: 2^25 workgroups would be more
    threads than a launch has"""
    slots, n = 1 << 25, 4097
    model = Model(1, 40, 1, 32, 16, True, 2, slots)
    rng = np.random.default_rng(1)
    at = np.r_[0:3, 65535:65538, (1 << 24) - 1:(1 << 24) + 2, slots - 2:slots]
    model.tables[0, at] = rng.permutation(40)[:len(at)]
    model.refs[:] = np.bincount(model.tables[0, at], minlength=40)
    pages = Pages(model)
    to, source = np.full(n, -1), np.full(n, 99)
    for i, length in ((4096, slots * 32), (7, (1 << 29) + 1), (0, 33)):
        to[:], source[:] = -1, 99
        to[i], source[i] = 1, 0
        lengths = np.full(n, length)
        assert pages.fork(to, source, lengths) == 0
        held = -(-length // 32)
        model.tables[1, :held], model.tables[1, held:] = model.tables[0, :held], -1
        model.refs[:] = np.bincount(model.tables[model.tables >= 0], minlength=40)
        pages.same()


def test_a_refused_fork_shows_in_a_status_of_its_own():
    """a fork and a reserve queued one after the other, the fork's lists such as are refused: a word each tells both; one word would
    say that all is well, over a sequence that never got the pages"""
    pages = Pages(filled(np.random.default_rng(2), 1, 1, 32, 16, True, [70, 0, 0]))
    model, lib = pages.m, pages.lib
    to, source, starts, ends, status = ints([1, 2]), ints([0, 3]), ints([70, 70]), ints([71, 71]), ints([77, 77])
    for words in ((0, 4), (0, 0)):
        check(lib.hk_pages_fork(pages.ref, to.ptr, source.ptr, starts.ptr, 2, status.ptr.value + words[0], None))
        check(lib.hk_pages_reserve(pages.ref, to.ptr, starts.ptr, ends.ptr, 2, status.ptr.value + words[1], pages.space.ptr, pages.need, None))
        assert status.numpy().tolist() == ([-1, 0] if words[1] else [0, 0])
        assert model.reserve([1, 2], [70, 70], [71, 71]) == 0
        assert (model.tables[1:, :2] < 0).all()
        pages.same()
