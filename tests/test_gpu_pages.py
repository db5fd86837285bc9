"""hk_pages_*: the tables, counts and pools after calls equal to the NumPy model's, the attention within the derived bound of
its float64 form."""
import ctypes

import numpy as np
import pytest

from gpu_lib import Dev, check, hip, hip_check, upload
from pages_lib import Model, Pages, at, filled, ints, within
from paths import package

pytestmark = pytest.mark.gpu

# layers, pages, kv heads, page size, head size, float16, sequences, table size
SHAPES = [(2, 40, 2, 32, 16, True, 6, 9), (1, 30, 3, 64, 48, False, 5, 8), (3, 50, 1, 128, 96, True, 7, 7),
          (1, 37, 2, 256, 32, False, 9, 5), (2, 14, 2, 32, 16, True, 6, 9)]  # (the last: calls that lack pages)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("seed", range(3))
def test_calls_in_turn_follow_the_model(shape, seed):
    rng = np.random.default_rng(100 * seed + shape[1])
    model = Model(*shape, rng=rng)
    pages, n, most = Pages(model), shape[6], shape[3] * shape[7]
    lengths = np.zeros(n, dtype=int)
    for _ in range(40):
        kind = rng.choice(["reserve", "reserve", "fork", "free", "compact"])
        some = rng.permutation(n)[:rng.integers(1, n + 1)].tolist()
        if kind == "reserve":
            starts = [int(lengths[s]) for s in some]
            ends = [min(most, a + int(rng.choice([0, 1, 1, 7, 40, 100, 300]))) for a in starts]
            got, want = pages.reserve(some, starts, ends), model.reserve(some, starts, ends)
            assert got == want
            if want == 0:
                layer = int(rng.integers(shape[0]))
                rows = [(s, p) for s, a, b in zip(some, starts, ends) for p in range(a, b)]
                if rows:
                    k, v = rng.standard_normal((2, len(rows), model.nkv * model.hs)).astype(np.float32)
                    for x in (pages, model):
                        x.append(layer, k, v, [s for s, _ in rows], [p for _, p in rows])
                for s, b in zip(some, ends):
                    lengths[s] = b
        elif kind == "fork":
            source = rng.integers(0, n, len(some)).tolist()
            cut = [int(rng.integers(0, lengths[f] + 1)) if rng.random() < 0.4 else int(lengths[f]) for f in source]
            assert pages.fork(some, source, cut) == model.fork(some, source, cut) == 0
            lengths[some] = cut
        elif kind == "free":
            kept = [int(rng.integers(0, lengths[s] + 1)) if rng.random() < 0.5 else 0 for s in some]
            for x in (pages, model):
                x.free(some, kept)
            lengths[some] = kept
        else:
            assert pages.compact() == model.compact()
        pages.same()


def test_lists_that_are_not_taken_change_nothing():
    rng = np.random.default_rng(5)
    model = filled(rng, 2, 2, 32, 16, True, [70, 33, 0, 10])
    pages, most = Pages(model), model.slots * model.page
    for seqs, starts, ends in (([0, 0], [70, 70], [71, 71]), ([4], [0], [1]), ([1, 2], [33, -1], [34, 5]),
                               ([1], [33], [most + 1]), ([1], [most + 1], [most + 1])):
        assert pages.reserve(seqs, starts, ends) == model.reserve(seqs, starts, ends) == -1
        pages.same()
    for to, source, lengths in (([2, 2], [0, 1], [5, 5]), ([4], [0], [5]), ([2], [4], [5]), ([2], [-1], [5]), ([2], [0], [-1]),
                                ([2], [0], [most + 1])):
        assert pages.fork(to, source, lengths) == model.fork(to, source, lengths) == -1
        pages.same()
    # all or nothing: the second entry lacks pages
    assert pages.reserve([1, 2], [33, 0], [64, most]) == model.reserve([1, 2], [33, 0], [64, most]) > 0
    pages.same()
    # negative sequences are passed over, whatever stands beside them
    assert pages.reserve([-1, 2, -5], [9999999, 0, -7], [0, 1, 3]) == model.reserve([-1, 2, -5], [9999999, 0, -7], [0, 1, 3]) == 0
    pages.same()
    assert pages.fork([-1, 3], [99, 0], [-4, 40]) == model.fork([-1, 3], [99, 0], [-4, 40]) == 0
    pages.same()
    # a sequence past the tables, and one listed twice: the smaller number holds
    for x in (pages, model):
        x.free([99, 0, -1, 0], [0, 64, 0, 33])
    pages.same()
    for x in (pages, model):
        x.free([1, 3])
    pages.same()


def test_beams_that_change_places():
    rng = np.random.default_rng(6)
    model = filled(rng, 1, 1, 32, 16, False, [100, 64, 33, 7, 0])
    pages = Pages(model)
    for to, source, lengths in (([0, 1, 2, 3], [1, 0, 3, 3], [64, 100, 7, 7]), ([0, 1, 2, 3, 4], [4, 4, 1, 1, 1], [0, 0, 100, 50, 64]),
                                ([2], [2], [40])):
        assert pages.fork(to, source, lengths) == model.fork(to, source, lengths) == 0
        pages.same()
    # both read the page: both part from it, and it is free then
    assert pages.reserve([2, 3], [40, 50], [41, 51]) == model.reserve([2, 3], [40, 50], [41, 51]) == 0
    pages.same()
    assert (model.refs >= 0).all()


@pytest.mark.parametrize("seqs, slots, page, n_pages", [(8192, 3, 32, 9000), (1000, 70, 64, 40000), (3, 9000, 32, 20000)])
def test_many_sequences_and_pages(seqs, slots, page, n_pages):
    """lists, tables and pools of more than one batch"""
    rng = np.random.default_rng(seqs)
    model = Model(1, n_pages, 1, page, 16, True, seqs, slots)
    model.keys[:] = np.arange(n_pages, dtype=np.float32)[None, :, None, None, None] / 64  # (a page's rows name it)
    pages = Pages(model)
    order = rng.permutation(seqs).tolist()
    half = [s for s in order if s % 2]
    ends = [int(rng.integers(0, min(slots * page, n_pages * page // seqs) + 1)) for _ in order]
    assert pages.reserve(order, [0] * seqs, ends) == model.reserve(order, [0] * seqs, ends) == 0
    pages.same()
    for x in (pages, model):
        x.free(half)
    pages.same()
    assert pages.compact() == model.compact()
    pages.same()
    lengths = dict(zip(order, ends))
    source = [s - 1 for s in half]
    cut = [lengths[s] for s in source]
    assert pages.fork(half, source, cut) == model.fork(half, source, cut) == 0
    pages.same()
    after = [min(slots * page, c + 1) for c in cut]
    got = pages.reserve(half, cut, after)
    assert got == model.reserve(half, cut, after)
    pages.same()


@pytest.mark.parametrize("nkv, hs, page, half", [(2, 16, 32, True), (3, 48, 64, False), (1, 256, 128, True), (8, 128, 256, False)])
def test_rows_that_are_dropped_rounded_and_padded(nkv, hs, page, half):
    rng = np.random.default_rng(nkv * hs)
    model = filled(rng, 2, nkv, page, hs, half, [page + 3, 5, 0])
    pages = Pages(model)
    seqs, positions = [0, 1, 2, 0, -1, 3, 1, 1, 0], [page + 2, 4, 0, 0, 0, 0, model.slots * page, -1, 2 * page]
    k = rng.standard_normal((9, nkv * hs)).astype(np.float32)
    v = rng.standard_normal((9, nkv * hs)).astype(np.float32)
    # halves between two float16 values, the largest ones, denormals, what is not finite
    k[0, :8] = [1 + 2 ** -11, 1 + 3 * 2 ** -11, 65504, 65519.996, 2 ** -24, 2 ** -25, 3 * 2 ** -26, -(2 ** -25)]
    k[3, :4] = [np.inf, -np.inf, 65520, 1e30]
    for pad in (0, 12):
        pages.append(1, k, v, seqs, positions, pad)
        model.append(1, k, v, seqs, positions)
        pages.same()
    pages.append(0, k[:2], v[:2], None, [1, 2])  # (no list: row i is sequence i)
    model.append(0, k[:2], v[:2], [0, 1], [1, 2])
    pages.same()


# query heads, kv heads, head size: every head size, groups of one to 32, odd ones
HEADS = [(4, 2, 16), (10, 5, 32), (6, 6, 48), (8, 8, 64), (12, 4, 96), (8, 2, 128), (7, 1, 128), (4, 2, 256), (32, 1, 64),
         (9, 1, 32), (17, 1, 16), (24, 2, 128), (32, 1, 256)]


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("nh, nkv, hs", HEADS)
def test_attention_at_lengths_where_it_can_go_wrong(nh, nkv, hs, half):
    rng = np.random.default_rng(nh * hs)
    lengths = [1, 31, 32, 33, 0, 127, 128, 129, 300, 513, 1030, 2]
    model = filled(rng, 2, nkv, 64, hs, half, lengths)
    # what lies behind the rows' ends, and in pages that none of them names
    for s, n in enumerate(lengths):
        for pool in (model.keys, model.values):
            if n % 64:
                pool[:, model.tables[s, n // 64], :, n % 64:] = [np.nan, np.inf, -np.inf][s % 3]
    model.values[:, model.refs == 0] = np.nan
    pages = Pages(model)
    seqs = rng.permutation(len(lengths))
    lens = np.asarray(lengths)[seqs].tolist()
    q = (1.5 * rng.standard_normal((len(lens), nh * hs))).astype(np.float32)
    got = pages.attention(1, q, seqs.tolist(), lens, nh, pad=8)
    within(got, model, 1, q, seqs.tolist(), lens, nh)
    assert (got[lens.index(0)] == 0).all()
    # one at a time (cut into pieces by its own length alone)
    for i in (lens.index(1030), lens.index(33)):
        alone = pages.attention(1, q[i:i + 1], [int(seqs[i])], [lens[i]], nh, longest=1030)
        within(alone, model, 1, q[i:i + 1], [int(seqs[i])], [lens[i]], nh)


@pytest.mark.parametrize("page", [32, 128, 256])
@pytest.mark.parametrize("half", [False, True])
def test_pages_of_every_size_and_no_list(page, half):
    rng = np.random.default_rng(page)
    lengths = [page - 1, page, page + 1, 5 * page + 7, 1]
    model = filled(rng, 1, 2, page, 64, half, lengths)
    pages = Pages(model)
    q = rng.standard_normal((5, 8 * 64)).astype(np.float32)
    within(pages.attention(0, q, None, lengths, 8), model, 0, q, None, lengths, 8)
    # longer launches than any row needs
    within(pages.attention(0, q, None, lengths, 8, longest=model.slots * page), model, 0, q, None, lengths, 8)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("rows", [63, 64, 65, 130, 256, 257, 700])
def test_many_rows(rows, half):
    """launches that plan their pieces from up to 256 rows' lengths, and ones of more; empty, short and long rows, some that
    cannot be, over the pages of a few sequences"""
    rng = np.random.default_rng(rows)
    held = [3000, 700, 64]
    model = filled(rng, 1, 2, 32, 32, half, held)
    pages = Pages(model)
    seqs = rng.integers(0, 3, rows)
    lengths = np.array([int(rng.integers(0, min(held[s], 200) + 1)) for s in seqs])
    for i in (0, rows // 2, rows - 1):  # the long ones, at the lists' ends
        seqs[i], lengths[i] = 0, 3000 - i
    seqs[1], seqs[2], lengths[3] = -1, 3, 3001  # (no sequence, none such, past `longest`)
    q = rng.standard_normal((rows, 6 * 32)).astype(np.float32)
    got = pages.attention(0, q, seqs.tolist(), lengths.tolist(), 6, longest=3000)
    wrong = [i for i in (2, 3) if lengths[i] > 0]
    assert np.isnan(got[wrong]).all() and (got[1] == 0).all()
    keep = np.array([i for i in range(rows) if i not in (2, 3)])
    within(got[keep], model, 0, q[keep], seqs[keep].tolist(), lengths[keep].tolist(), 6)


def test_pieces_of_more_pages_than_a_wave_looks_up_at_once():
    """more rows than are planned for, so many heads that a row is one piece: 9000 positions of one sequence to a workgroup"""
    rng = np.random.default_rng(12)
    model = filled(rng, 1, 64, 32, 16, True, [9000])
    pages = Pages(model)
    lengths = [9000, 8999, 8193, 8192] + [int(n) for n in rng.integers(1, 40, 296)]
    q = rng.standard_normal((300, 64 * 16)).astype(np.float32)
    got = pages.attention(0, q, [0] * 300, lengths, 64)
    within(got, model, 0, q, [0] * 300, lengths, 64)


def test_a_turn_of_one_sequence():
    """the tokens of a turn as rows one position apart, and a fork's rows beside them"""
    rng = np.random.default_rng(1)
    model = filled(rng, 1, 2, 32, 128, True, [700, 0])
    pages = Pages(model)
    assert pages.fork([1], [0], [650]) == model.fork([1], [0], [650]) == 0
    seqs, lengths = [0] * 20 + [1] * 3, list(range(681, 701)) + [1, 640, 650]
    q = rng.standard_normal((23, 8 * 128)).astype(np.float32)
    within(pages.attention(0, q, seqs, lengths, 8), model, 0, q, seqs, lengths, 8)


@pytest.mark.parametrize("half", [False, True])
def test_rows_that_have_no_attention(half):
    rng = np.random.default_rng(2)
    model = filled(rng, 1, 2, 32, 64, half, [100, 700, 64, 10])
    kept = model.tables[1, 9]
    pages = Pages(model)
    seqs, lengths = [0, 1, -1, 4, 2, 3, 0, 1, 3], [100, 700, 50, 10, 701, 0, 129, 300, -5]
    q = rng.standard_normal((9, 4 * 64)).astype(np.float32)
    for lost in (-1, model.pages, 1 << 30, -7):
        model.tables[1, 9] = lost  # (positions 288..319 of sequence 1)
        hip_check(hip().hipMemcpy(pages.dev["tables"].ptr, ctypes.c_void_p(model.tables.ctypes.data), model.tables.nbytes, 1))
        got = pages.attention(0, q, seqs, lengths, 4, longest=700)
        for i in (1, 3, 4, 6, 7):  # no page; no such sequence; longer than the launch; past the sequence's pages; no page
            assert np.isnan(got[i]).all(), i
        for i in (2, 5, 8):
            assert (got[i] == 0).all()
        within(got[:1], model, 0, q[:1], seqs[:1], lengths[:1], 4)
    model.tables[1, 9] = kept


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("length", [40, 1500])
def test_numbers_that_are_not_finite_stay_in_their_rows(half, length):
    rng = np.random.default_rng(3)
    model = filled(rng, 1, 2, 32, 64, half, [length] * 5)
    q = rng.standard_normal((5, 4 * 64)).astype(np.float32)
    q[1, 3] = np.nan   # query head 0 of row 1
    q[2, 64] = np.inf  # query head 1 of row 2
    model.keys[0, model.tables[3, 1], 0, 5, 7] = np.nan   # kv head 0 of row 3
    model.values[0, model.tables[4, 0], 1, 2, 9] = np.inf  # kv head 1's channel 9 of row 4
    got = Pages(model).attention(0, q, None, [length] * 5, 4)
    lost = np.zeros(got.shape, dtype=bool)
    lost[1, 0] = lost[2, 1] = lost[3, :2] = lost[4, 2:, 9] = True
    assert np.isnan(got[1, 0]).all() and np.isnan(got[2, 1]).all() and np.isnan(got[3, :2]).all()
    assert not np.isfinite(got[4, 2:, 9]).any()
    assert np.isfinite(got[~lost]).all()
    model.keys[0, model.tables[3, 1], 0, 5, 7] = 0
    model.values[0, model.tables[4, 0], 1, 2, 9] = 0
    q[1, 3] = q[2, 64] = 0
    want, off = model.attention(0, q, None, [length] * 5, 4)
    assert (np.abs(got - want) <= off)[0].all()


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("scale", [1e-40, 1e-30, 1e-6, 30.0, 1e4])
def test_queries_of_any_size(half, scale):
    """scores next to nothing, and so large that one position takes all"""
    rng = np.random.default_rng(4)
    lengths = [3, 200, 900]
    model = filled(rng, 1, 1, 32, 64, half, lengths)
    if half:
        model.keys[0, :, :, :, 5] *= 20000  # (the largest float16 values beside ordinary ones)
    q = (scale * rng.standard_normal((3, 4 * 64))).astype(np.float32)
    q.reshape(3, 4, 64)[:, :, 5] *= 1e-4
    within(Pages(model).attention(0, q, None, lengths, 4), model, 0, q, None, lengths, 4)


@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("keys, values", [(1e-6, 1.0), (1.0, 1e-6), (1e-6, 1e-6), (1.0, 3e-8)])
def test_keys_and_values_next_to_nothing(half, keys, values):
    """(in float16: denormals) against queries that make their scores count"""
    rng = np.random.default_rng(13)
    lengths = [3, 200, 900]
    model = filled(rng, 1, 1, 32, 64, half, lengths)
    model.keys[:] = model.keys * np.float32(keys)
    model.values[:] = model.values * np.float32(values)
    q = (rng.standard_normal((3, 4 * 64)) / keys).astype(np.float32)
    within(Pages(model).attention(0, q, None, lengths, 4), model, 0, q, None, lengths, 4)


@pytest.mark.parametrize("half", [False, True])
def test_a_score_that_grows(half):
    """every block of positions with scores far above the last one's, and far below"""
    lengths, hs = [1200, 1200], 32
    rng = np.random.default_rng(7)
    model = filled(rng, 1, 1, 32, hs, half, lengths)
    for s, sign in ((0, 1.0), (1, -1.0)):
        for b in range(38):
            model.keys[0, model.tables[s, b], 0] = sign * b * 3.0 + 0.1 * rng.standard_normal((32, hs))
    q = np.full((2, 2 * hs), 0.5, dtype=np.float32)
    within(Pages(model).attention(0, q, None, lengths, 2), model, 0, q, None, lengths, 2)


def test_large_values_behind_scores_that_grow():
    """values near float32's largest: none is weighted by more than 1 on the way, however the scores grow from block to block"""
    rng = np.random.default_rng(14)
    model = filled(rng, 1, 1, 32, 32, False, [1200])
    for b in range(38):
        model.keys[0, model.tables[0, b], 0] = b * 0.7 + 0.1 * rng.standard_normal((32, 32))
    model.values[:] = model.values * np.float32(1e36)
    q = np.full((1, 2 * 32), 0.5, dtype=np.float32)
    within(Pages(model).attention(0, q, None, [1200], 2), model, 0, q, None, [1200], 2)


def test_keys_of_minus_infinity_have_no_weight():
    """in a float32 cache, where the query's value is above 0: the other rows' scores stand"""
    rng = np.random.default_rng(15)
    model = filled(rng, 1, 1, 32, 32, False, [100])
    q = np.abs(rng.standard_normal((1, 2 * 32))).astype(np.float32) + np.float32(0.1)
    model.keys[0, model.tables[0, 1], 0, 3, 5] = -np.inf  # position 35
    got = Pages(model).attention(0, q, None, [100], 2)
    model.keys[0, model.tables[0, 1], 0, 3] = -1e4
    within(got, model, 0, q, None, [100], 2)


@pytest.mark.parametrize("half", [False, True])
def test_a_long_context(half):
    rng = np.random.default_rng(8)
    lengths = [20011, 9, 33000]
    model = filled(rng, 1, 1, 128, 64, half, lengths)
    q = rng.standard_normal((3, 4 * 64)).astype(np.float32)
    within(Pages(model).attention(0, q, None, lengths, 4), model, 0, q, None, lengths, 4)


def test_offsets_past_32_bits():
    """the last pages and layer of pools of 5 GB: their rows lie past 2^32 bytes and 2^31 values"""
    lib, h, rng = package().library(), hip(), np.random.default_rng(9)
    layers, n_pages, nkv, page, hs = 2, 5000, 8, 256, 128
    size = layers * n_pages * nkv * page * hs * 2
    assert size // 2 > 1 << 31
    pools = []
    for _ in range(2):
        p = ctypes.c_void_p()
        hip_check(h.hipMalloc(ctypes.byref(p), ctypes.c_size_t(size)))
        pools.append(p)
    small = filled(rng, 1, nkv, page, hs, True, [600], spare=0)  # (three pages: the same rows, in a model of their own)
    small.tables[0, :3] = [0, 1, 2]
    tables = np.full((1, 4), -1, dtype=np.int32)
    tables[0, :3] = [n_pages - 2, 1, n_pages - 3]
    refs = np.zeros(n_pages, dtype=np.int32)
    refs[tables[0, :3]] = 1
    td, rd = upload(tables), upload(refs)
    c = package().HkPages(keys=pools[0].value, values=pools[1].value, tables=td.ptr.value, refs=rd.ptr.value, n_layers=layers,
                          n_pages=n_pages, n_kv_heads=nkv, page_size=page, head_size=hs, half=1, n_seqs=1, table_size=4)
    ref = ctypes.byref(c)
    k, v = (x.astype(np.float32).reshape(600, -1) for x in small.rows(0, 0, 600))
    q = rng.standard_normal((1, 16 * hs)).astype(np.float32)
    kd, vd, qd, out = upload(k), upload(v), upload(q), Dev((1, 16 * hs), np.float32)
    seqs, positions, lengths, start = ints([0] * 600), ints(range(600)), ints([600]), ints([0])
    need = lib.hk_pages_attention_workspace(ref, 16, 1, 600)
    more = lib.hk_pages_workspace(ref)
    space = Dev(max(need, more, 1), np.uint8)
    check(lib.hk_pages_append(ref, 1, kd.ptr, vd.ptr, nkv * hs, seqs.ptr, positions.ptr, 600, None))

    def attend():
        check(lib.hk_pages_attention(out.ptr, qd.ptr, ref, 1, 16, 16 * hs, 16 * hs, start.ptr, lengths.ptr, 1, 600, space.ptr, need, None))
        return out.numpy().reshape(1, 16, hs)

    got = attend()
    within(got, small, 0, q, None, [600], 16)
    used = ints([0])
    check(lib.hk_pages_compact(ref, used.ptr, space.ptr, more, None))
    assert used.numpy()[0] == 3 and td.numpy()[0].tolist() == [2, 1, 0, -1]
    np.testing.assert_array_equal(attend(), got)
    for p in pools:
        hip_check(h.hipFree(p))


def test_steps_replayed_from_a_graph():
    """a step of three conversations (room, rows, attention) captured once and replayed, the lists changing between, with eager
    calls of the same cache beside it"""
    lib, h, rng = package().library(), hip(), np.random.default_rng(10)
    nh, nkv, hs, page = 8, 2, 64, 32
    model = filled(rng, 2, nkv, page, hs, True, [30, 95, 0], spare=12, slots=8)
    pages = Pages(model)
    lens = [30, 95, 0]
    stream, graph, run = ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_void_p()
    hip_check(h.hipStreamCreate(ctypes.byref(stream)))
    bufs = {name: Dev((3, n), np.float32) for name, n in (("k", nkv * hs), ("v", nkv * hs), ("q", nh * hs), ("out", nh * hs))}
    seqs, starts, ends, status = ints([0, 1, 2]), ints([0] * 3), ints([0] * 3), ints([0])
    need = lib.hk_pages_attention_workspace(pages.ref, nh, 3, 256)
    space = Dev(max(1, need), np.uint8)
    hip_check(hip().hipDeviceSynchronize())
    hip_check(h.hipStreamBeginCapture(stream, 2))
    check(lib.hk_pages_reserve(pages.ref, seqs.ptr, starts.ptr, ends.ptr, 3, status.ptr, pages.space.ptr, pages.need, stream))
    for layer in range(2):
        check(lib.hk_pages_append(pages.ref, layer, bufs["k"].ptr, bufs["v"].ptr, nkv * hs, seqs.ptr, starts.ptr, 3, stream))
        check(lib.hk_pages_attention(bufs["out"].ptr, bufs["q"].ptr, pages.ref, layer, nh, nh * hs, nh * hs, seqs.ptr, ends.ptr, 3,
                                     256, space.ptr, need, stream))
    hip_check(h.hipStreamEndCapture(stream, ctypes.byref(graph)))
    hip_check(h.hipGraphInstantiate(ctypes.byref(run), graph, None, None, 0))

    def put(dev, x):
        x = np.ascontiguousarray(x, dtype=dev.dtype)
        hip_check(h.hipMemcpy(dev.ptr, ctypes.c_void_p(x.ctypes.data), dev.nbytes, 1))

    for step in range(6):
        order = rng.permutation(3)
        k, v = rng.standard_normal((2, 3, nkv * hs)).astype(np.float32)
        q = rng.standard_normal((3, nh * hs)).astype(np.float32)
        a = [lens[s] for s in order]
        for dev, x in ((bufs["k"], k), (bufs["v"], v), (bufs["q"], q), (seqs, order), (starts, a), (ends, [n + 1 for n in a])):
            put(dev, x)
        hip_check(h.hipGraphLaunch(run, stream))
        hip_check(h.hipStreamSynchronize(stream))
        assert model.reserve(order.tolist(), a, [n + 1 for n in a]) == status.numpy()[0] == 0
        for layer in range(2):
            model.append(layer, k, v, order.tolist(), a)
        pages.same()
        got = bufs["out"].numpy().reshape(3, nh, hs)
        lengths = [n + 1 for n in a]
        within(got, model, 1, q, order.tolist(), lengths, nh)
        np.testing.assert_array_equal(got, pages.attention(1, q, order.tolist(), lengths, nh, longest=256))
        for s in range(3):
            lens[s] += 1
        if step == 2:  # the second conversation ends, and goes on from the first's beginning
            assert pages.fork([1], [0], [31]) == model.fork([1], [0], [31]) == 0
            lens[1] = 31
    hip_check(h.hipGraphExecDestroy(run))
    hip_check(h.hipGraphDestroy(graph))
    hip_check(h.hipStreamDestroy(stream))


def test_housekeeping_replayed_from_a_graph():
    """sequences ended, forked, given room and compacted by one captured graph, the lists changing between its replays"""
    lib, h, rng = package().library(), hip(), np.random.default_rng(16)
    model = filled(rng, 2, 2, 32, 16, False, [70, 40, 100, 0, 0, 33], spare=20, slots=8)
    pages, lens, n = Pages(model), [70, 40, 100, 0, 0, 33], 3
    lists = {name: ints([0] * n) for name in ("ended", "to", "source", "lengths", "ends")}
    status, used = ints([7, 7]), ints([7])
    stream, graph, run = ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_void_p()
    hip_check(h.hipStreamCreate(ctypes.byref(stream)))
    hip_check(h.hipDeviceSynchronize())
    hip_check(h.hipStreamBeginCapture(stream, 2))
    check(lib.hk_pages_free(pages.ref, lists["ended"].ptr, None, n, stream))
    check(lib.hk_pages_fork(pages.ref, lists["to"].ptr, lists["source"].ptr, lists["lengths"].ptr, n, status.ptr, stream))
    check(lib.hk_pages_reserve(pages.ref, lists["to"].ptr, lists["lengths"].ptr, lists["ends"].ptr, n, status.ptr.value + 4,
                               pages.space.ptr, pages.need, stream))
    check(lib.hk_pages_compact(pages.ref, used.ptr, pages.space.ptr, pages.need, stream))
    hip_check(h.hipStreamEndCapture(stream, ctypes.byref(graph)))
    hip_check(h.hipGraphInstantiate(ctypes.byref(run), graph, None, None, 0))
    for _ in range(5):
        order = rng.permutation(6).tolist()
        ended, to = order[:1] + [-1, -1], order[1:4]
        lens[ended[0]] = 0
        source = [int(rng.choice(6)) for _ in to]
        cut = [int(rng.integers(0, lens[f] + 1)) for f in source]
        ends = [min(256, a + int(rng.integers(1, 40))) for a in cut]
        for name, x in zip(lists, (ended, to, source, cut, ends)):
            x = np.asarray(x, dtype=np.int32)
            hip_check(h.hipMemcpy(lists[name].ptr, ctypes.c_void_p(x.ctypes.data), x.nbytes, 1))
        hip_check(h.hipGraphLaunch(run, stream))
        hip_check(h.hipStreamSynchronize(stream))
        model.free(ended)
        want = [model.fork(to, source, cut), model.reserve(to, cut, ends)]
        assert status.numpy().tolist() == want and want[0] == 0
        assert used.numpy()[0] == model.compact()
        pages.same()
        for s, a, b in zip(to, cut, ends):
            lens[s] = b if want[1] == 0 else a
        for x in (pages, model):  # an eager call between the replays
            x.free([order[5]], [lens[order[5]] // 2])
        lens[order[5]] //= 2
        pages.same()
    hip_check(h.hipGraphExecDestroy(run))
    hip_check(h.hipGraphDestroy(graph))
    hip_check(h.hipStreamDestroy(stream))


def test_two_streams_at_once():
    """two layers' attention on two streams, each with its own workspace: the results of the calls one after the other"""
    lib, h, rng = package().library(), hip(), np.random.default_rng(11)
    nh, hs, lengths = 8, 128, [5000, 17, 2500]
    model = filled(rng, 2, 2, 64, hs, True, lengths)
    pages = Pages(model)
    q = rng.standard_normal((3, nh * hs)).astype(np.float32)
    want = [pages.attention(layer, q, None, lengths, nh) for layer in range(2)]
    need = lib.hk_pages_attention_workspace(pages.ref, nh, 3, 5000)
    qd, lens, work = upload(q), ints(lengths), []
    for layer in range(2):
        stream = ctypes.c_void_p()
        hip_check(h.hipStreamCreate(ctypes.byref(stream)))
        work.append((layer, stream, Dev((3, nh * hs), np.float32), Dev(max(1, need), np.uint8)))
    hip_check(h.hipDeviceSynchronize())
    for _ in range(5):
        for layer, stream, out, space in work:
            check(lib.hk_pages_attention(out.ptr, qd.ptr, pages.ref, layer, nh, nh * hs, nh * hs, None, lens.ptr, 3, 5000, space.ptr,
                                         need, stream))
    for layer, stream, out, _ in work:
        hip_check(h.hipStreamSynchronize(stream))
        np.testing.assert_array_equal(out.numpy().reshape(3, nh, hs), want[layer])
        hip_check(h.hipStreamDestroy(stream))
