"""hk_matmul_four against its definition in float64, and a decode step of several conversations over the cache in pages with
4-bit matrices."""
import numpy as np
import pytest

from gpu_lib import Dev, check, quantize_x, upload
from pages_lib import Pages, filled
from paths import package

pytestmark = pytest.mark.gpu


def columns(w, k):
    """the 4-bit values of packed rows, one column at a time, int [rows][k]"""
    c = np.arange(k)
    byte, high = 64 * (c // 128) + 16 * (c // 4 % 4) + 4 * (c // 32 % 4) + c % 4, c // 16 % 2
    four = w[:, byte].astype(np.int64) >> 4 * high & 15
    return np.where(four > 7, four - 16, four)


def product(xq, xs, w, ws, k, bias, group):
    """(y, bound) in float64: the group sums are exact, a group's scaled sum takes two roundings of 2^-24 and the scales'
    product one, and a sum of n of them at most n + 3"""
    m, rows, n = len(xq), len(w), k // 32
    x = (xq.astype(np.int64) - bias).reshape(m, n, 32)
    sums = np.einsum("tgi,rgi->trg", x, columns(w, k).reshape(rows, n, 32)).astype(np.float64)
    parts = sums * np.repeat(ws.astype(np.float64), group // 32, axis=1)[:, :n] * xs.astype(np.float64)[:, None]
    return parts.sum(-1), np.abs(parts).sum(-1) * (n + 6) * 2.0 ** -24


def four(xq, xs, w, ws, rows, k, bias, group):
    m = len(xq)
    y = upload(np.full((m, rows), 7.0, dtype=np.float32))
    args = [upload(a) for a in (xq, xs, w, ws)]
    check(package().library().hk_matmul_four(y.ptr, *(a.ptr for a in args), m, rows, k, bias, group,
                                             int(ws.dtype == np.float16), None))
    got = y.numpy()
    del args
    return got


def inputs(rng, m, rows, k, bias, group, half):
    most = 63 if bias else 127
    xq = (rng.integers(-most, most + 1, (m, k)) + bias).astype(np.int8)
    xs = rng.uniform(0.001, 0.1, (m, k // 32)).astype(np.float32)
    w, ws = package().quantize_four(rng.standard_normal((rows, k)), group, half)
    return xq, xs, w, ws


@pytest.mark.parametrize("group, half", [(32, False), (32, True), (64, False), (64, True), (128, False), (128, True)])
@pytest.mark.parametrize("rows, k", [(1, 32), (3, 96), (5, 128), (64, 288), (67, 768), (129, 1056), (33, 8224), (17, 18944)])
@pytest.mark.parametrize("m", [1, 2, 5, 16, 33])
def test_products_at_sizes_where_they_can_go_wrong(rows, k, m, group, half):
    rng = np.random.default_rng(rows * k + m)
    for bias in (0, 64):
        xq, xs, w, ws = inputs(rng, m, rows, k, bias, group, half)
        want, off = product(xq, xs, w, ws, k, bias, group)
        got = four(xq, xs, w, ws, rows, k, bias, group)
        assert (np.abs(got - want) <= off).all(), np.abs(got - want).max()


@pytest.mark.parametrize("m", [3, 4, 6, 7, 8, 9, 12, 15, 17, 24, 31, 32, 47, 48, 49, 63, 64, 65, 100, 130])
def test_any_number_of_tokens(m):
    rng = np.random.default_rng(m)
    for rows, k in ((100, 416), (1500, 1024), (20, 40000)):
        xq, xs, w, ws = inputs(rng, m, rows, k, 64, 32, False)
        want, off = product(xq, xs, w, ws, k, 64, 32)
        assert (np.abs(four(xq, xs, w, ws, rows, k, 64, 32) - want) <= off).all()


@pytest.mark.parametrize("m", [1, 2])
@pytest.mark.parametrize("k", [512, 544, 1024, 1056, 2048, 2080, 4096, 4128, 8192, 8224, 16384, 16416, 32768, 32800])
def test_rows_of_every_length(m, k):
    """one token and two, at the lengths between the kernel's shapes; more rows than a launch has places for at the shorter"""
    rng = np.random.default_rng(k)
    rows = 70001 if k < 600 else 9001 if k < 1100 else 37
    xq, xs, w, ws = inputs(rng, m, rows, k, 64, 64, True)
    want, off = product(xq, xs, w, ws, k, 64, 64)
    assert (np.abs(four(xq, xs, w, ws, rows, k, 64, 64) - want) <= off).all()


@pytest.mark.parametrize("group, half", [(32, False), (32, True), (64, False), (64, True), (128, False), (128, True)])
@pytest.mark.parametrize("m, rows, k", [(600, 411, 416), (600, 833, 416), (70, 2051, 1056), (130, 2739, 96), (49, 4101, 288), (40, 8209, 160),
                                        (20, 4111, 4128), (31, 8195, 4160), (16, 2050, 2112), (16, 4099, 1056), (32, 4105, 1312)])
def test_many_rows_of_many_tokens(m, rows, k, group, half):
    """the rows that a workgroup takes go by the tokens too: 16, 32 and 64 of them, with rows, tokens and columns left over"""
    rng = np.random.default_rng(m * rows + k)
    xq, xs, w, ws = inputs(rng, m, rows, k, 64, group, half)
    got = four(xq, xs, w, ws, rows, k, 64, group)
    some = np.unique(np.r_[np.arange(70), rng.integers(0, rows, 120), np.arange(rows - 70, rows)])  # (of the rows: the oracle's time)
    want, off = product(xq, xs, w[some], ws[some], k, 64, group)
    assert (np.abs(got[:, some] - want) <= off).all()
    alone = four(xq[m // 2:m // 2 + 1], xs[m // 2:m // 2 + 1], w, ws, rows, k, 64, group)  # (all the rows, by another kernel)
    _, off = product(xq[m // 2:m // 2 + 1], xs[m // 2:m // 2 + 1], w, ws, k, 64, group)
    assert (np.abs(got[m // 2] - alone[0]) <= 2 * off[0]).all()


def test_every_pair_of_values():
    """all 4-bit values against all activations at the ends of their range"""
    rows, k = 16, 160
    vals = np.tile(np.arange(-8, 8), (rows, k // 16))
    vals = (vals + np.arange(rows)[:, None] + 8) % 16 - 8
    q = np.zeros((rows, 256), dtype=np.int64)
    q[:, :k] = vals
    part = (q & 15).reshape(rows, 2, 4, 2, 4, 4).transpose(3, 0, 1, 4, 2, 5)
    w = (part[0] | part[1] << 4).astype(np.uint8).reshape(rows, -1)
    np.testing.assert_array_equal(columns(w, 256), q)
    ws = np.ones((rows, 8), dtype=np.float32)
    ws[:, 5:] = 0
    for x in (-128, -127, 127, 0):
        for m in (1, 20):
            xq = np.full((m, k), x, dtype=np.int8)
            got = four(xq, np.ones((m, 5), dtype=np.float32), w, ws, rows, k, 0, 32)
            np.testing.assert_array_equal(got, np.tile((vals * x).sum(-1), (m, 1)).astype(np.float32))


@pytest.mark.parametrize("m, rows, k", [(3, 40, 768), (5, 40, 2048), (20, 40, 2048), (17, 40, 768), (40, 70, 1024), (6, 40, 8192)])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_a_scale_that_is_not_finite_concerns_its_token_alone(m, rows, k, bad):
    rng = np.random.default_rng(m + k)
    xq, xs, w, ws = inputs(rng, m, rows, k, 64, 64, False)
    want = four(xq, xs, w, ws, rows, k, 64, 64)
    for t in {0, m // 2, m - 1}:
        other = xs.copy()
        other[t, k // 64] = bad
        y = four(xq, other, w, ws, rows, k, 64, 64)
        assert not np.isfinite(y[t]).any()
        keep = np.arange(m) != t
        np.testing.assert_array_equal(y[keep], want[keep])


@pytest.mark.parametrize("m, rows, k", [(1, 300, 4096), (1, 40, 9000 // 32 * 32), (16, 300, 4096), (7, 100, 768), (20, 300, 2048), (40, 70, 1024),
                                        (5, 40, 8192)])
def test_products_replayed_from_a_graph(m, rows, k):
    import ctypes
    from gpu_lib import hip, hip_check
    h, rng = hip(), np.random.default_rng(m + k)
    stream, graph, run = ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_void_p()
    hip_check(h.hipStreamCreate(ctypes.byref(stream)))
    xq, xs, w, ws = inputs(rng, m, rows, k, 64, 32, True)
    args, y = [upload(a) for a in (xq, xs, w, ws)], Dev((m, rows), np.float32)
    hip_check(h.hipDeviceSynchronize())
    hip_check(h.hipStreamBeginCapture(stream, 2))
    check(package().library().hk_matmul_four(y.ptr, *(a.ptr for a in args), m, rows, k, 64, 32, 1, stream))
    hip_check(h.hipStreamEndCapture(stream, ctypes.byref(graph)))
    hip_check(h.hipGraphInstantiate(ctypes.byref(run), graph, None, None, 0))
    for _ in range(3):
        xq, xs, _, _ = inputs(rng, m, 1, k, 64, 32, True)
        for dev, x in zip(args, (xq, xs)):
            hip_check(h.hipMemcpy(dev.ptr, ctypes.c_void_p(x.ctypes.data), dev.nbytes, 1))
        hip_check(h.hipGraphLaunch(run, stream))
        hip_check(h.hipStreamSynchronize(stream))
        np.testing.assert_array_equal(y.numpy(), four(xq, xs, w, ws, rows, k, 64, 32))  # (an eager call between the replays)
        want, off = product(xq, xs, w, ws, k, 64, 32)
        assert (np.abs(y.numpy() - want) <= off).all()
    hip_check(h.hipGraphExecDestroy(run))
    hip_check(h.hipGraphDestroy(graph))
    hip_check(h.hipStreamDestroy(stream))


def test_a_step_of_conversations():
    """one layer of a decode step, as a program that answers several conversations makes it: quantized activations, q, k and v
    by 4-bit matrices, room and rows in the pages, attention, the output's product; against the same in float64 on the
    quantized numbers"""
    lib, pk, rng = package().library(), package(), np.random.default_rng(0)
    dim, nh, nkv, hs, page = 512, 8, 2, 64, 32
    lengths = [64, 31, 200, 7]
    n, width = len(lengths), nkv * hs
    model = filled(rng, 1, nkv, page, hs, False, lengths, spare=6)
    # the third goes on from the first three positions of the second as well
    pages = Pages(model)
    assert pages.fork([3], [1], [31]) == model.fork([3], [1], [31]) == 0
    lengths[3] = 31
    qkv, wo = pk.quantize_four(0.05 * rng.standard_normal((nh * hs + 2 * width, dim))), pk.quantize_four(
        0.05 * rng.standard_normal((dim, nh * hs)), 64, True)
    x = rng.standard_normal((n, dim)).astype(np.float32)
    xq, xs = quantize_x(x, 64)
    rows = four(xq, xs, *qkv, nh * hs + 2 * width, dim, 64, 32)
    want, off = product(xq, xs, *qkv, dim, 64, 32)
    assert (np.abs(rows - want) <= off).all()
    q, k, v = (np.ascontiguousarray(a) for a in np.split(rows, [nh * hs, nh * hs + width], axis=1))
    ends = [a + 1 for a in lengths]
    assert pages.reserve(list(range(n)), lengths, ends) == model.reserve(list(range(n)), lengths, ends) == 0
    pages.append(0, k, v, None, lengths)
    model.append(0, k, v, list(range(n)), lengths)
    pages.same()
    got = pages.attention(0, q, None, ends, nh)
    exact, off = model.attention(0, q, None, ends, nh)
    assert (np.abs(got - exact) <= off).all()
    aq, as_ = quantize_x(got.reshape(n, -1), 64)
    out = four(aq, as_, *wo, dim, nh * hs, 64, 64)
    want, off = product(aq, as_, *wo, nh * hs, 64, 64)
    assert (np.abs(out - want) <= off).all()
