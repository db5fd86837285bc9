"""hk_logprobs against NumPy in float64."""
import ctypes

import numpy as np
import pytest

from gpu_lib import Dev, check, hip, hip_check, upload
from paths import package

pytestmark = pytest.mark.gpu


def expected(x, given, top):
    x = x.astype(np.float64)
    m = x.max(-1, keepdims=True)
    with np.errstate(invalid="ignore"):
        e = np.exp(x - m)
        logz = np.log(e.sum(-1, keepdims=True))
        h = logz[:, 0] - np.where(e > 0, e * (x - m), 0).sum(-1) / e.sum(-1)
    order = np.argsort(-x, axis=-1, kind="stable")[:, :top]
    best = np.take_along_axis(x, order, -1)
    ids = np.where(best > -np.inf, order, -1)
    if ids.shape[1] < top:
        pad = ((0, 0), (0, top - ids.shape[1]))
        ids, best = np.pad(ids, pad, constant_values=-1), np.pad(best, pad, constant_values=-np.inf)
    logp = np.take_along_axis(x, given, -1) - m - logz if given is not None else None
    return logp, h, ids, best - m - logz


def run(x, given, top, stride=None, entropy=True, shift=0):
    """hk_logprobs on device copies; the logits start `shift` floats behind an aligned address"""
    lib = package().library()
    m, n = x.shape
    stride = stride or n
    wide = np.full(m * stride + shift, np.nan, dtype=np.float32)
    for i in range(m):
        wide[shift + i * stride:shift + i * stride + n] = x[i]
    xd = upload(wide)
    g = 0 if given is None else given.shape[1]
    gd = upload(given.astype(np.int32)) if g else None
    logp, ent = Dev((m, max(1, g)), np.float32), Dev(m, np.float32)
    ids, logps = Dev((m, max(1, top)), np.int32), Dev((m, max(1, top)), np.float32)
    need = lib.hk_logprobs_workspace(m, n, top)
    assert need >= 0
    space = Dev(max(1, need), np.uint8, np.full(max(1, need), 0xFF))
    check(lib.hk_logprobs(logp.ptr if g else None, ent.ptr if entropy else None, ids.ptr if top else None,
                          logps.ptr if top else None, ctypes.c_void_p(xd.ptr.value + 4 * shift), stride,
                          gd.ptr if g else None, g, m, n, top, space.ptr, need, None))
    return logp.numpy()[:, :g], ent.numpy(), ids.numpy()[:, :top], logps.numpy()[:, :top]


def agree(x, given, top, **how):
    """The bound: a log probability is x - m - log Z. Z is a sum of n positive terms, each off by 2^-22 (its exponential of a
    difference rounded once: 2^-24 |x - m|, where |x - m| < 20 for the terms that count) and summed in float32 runs of at
    most 2048 (2^-13 at the very worst, 2^-24 sqrt(2048) < 2^-18 as it happens): 2^-17 off at most as taken here; the result
    is rounded to float32 (2^-24 of its size). The entropy is two such sums, the second of terms below 20: 2^-12."""
    logp, h, ids, logps = run(x, given, top, **how)
    wl, wh, wi, wp = expected(x, given, top)
    np.testing.assert_array_equal(ids, wi)
    for got, want in ((logp, wl), (logps, wp)):
        if want is None or not got.size:
            continue
        infinite = np.isneginf(want)
        np.testing.assert_array_equal(np.isneginf(got), infinite)
        got, want = got[~infinite], want[~infinite]
        assert (np.abs(got - want) <= 2.0 ** -17 + 2.0 ** -23 * np.abs(want)).all()
    if how.get("entropy", True):
        assert (np.abs(h - wh) <= 2.0 ** -12 + 2.0 ** -22 * wh).all()


@pytest.mark.parametrize("m, n", [(1, 1), (1, 2), (3, 31), (2, 64), (5, 257), (1, 4096), (7, 1023), (2, 8193), (1, 32000),
                                  (33, 320), (3, 50257), (1, 128256), (2, 152064), (300, 515), (1, 262147)])
@pytest.mark.parametrize("top", [0, 1, 5, 32])
def test_rows(m, n, top):
    rng = np.random.default_rng(m * n + top)
    x = (rng.standard_normal((m, n)) * 3).astype(np.float32)
    given = rng.integers(0, n, (m, 1 + n % 3))
    agree(x, given, top)


@pytest.mark.parametrize("pad", [0, 1, 3, 64])
@pytest.mark.parametrize("shift", [0, 1, 2, 3])
def test_strides_and_alignment(pad, shift):
    rng = np.random.default_rng(pad + shift)
    x = (rng.standard_normal((4, 5003)) * 3).astype(np.float32)
    agree(x, rng.integers(0, 5003, (4, 2)), 7, stride=5003 + pad, shift=shift)


@pytest.mark.parametrize("order", ["up", "down", "equal", "few values", "one far", "two halves"])
@pytest.mark.parametrize("n", [40, 5000, 128256])
def test_orders_and_ties(order, n):
    """rows that the search for the largest finds hard: sorted either way, all equal, ties by the thousand"""
    rng = np.random.default_rng(n)
    x = np.zeros((2, n), dtype=np.float32)
    if order == "up":
        x[:] = np.linspace(-8, 8, n)
    elif order == "down":
        x[:] = np.linspace(8, -8, n)
    elif order == "few values":
        x[:] = rng.integers(-3, 3, (2, n))
    elif order == "one far":
        x[:, n // 3] = 80.0
    elif order == "two halves":
        x[:, n // 2:] = np.linspace(0, 3, n - n // 2)
    agree(x, rng.integers(0, n, (2, 3)), 32)


def test_banned_tokens():
    """logits of minus infinity: probability 0; fewer tokens left than alternatives asked for"""
    rng = np.random.default_rng(3)
    x = (rng.standard_normal((6, 3001)) * 2).astype(np.float32)
    x[rng.random(x.shape) < 0.5] = -np.inf
    x[1, 4:] = -np.inf
    x[1, 2] = 0.5
    x[2] = -np.inf
    x[2, 3000] = -200.0
    given = rng.integers(0, 3001, (6, 4))
    agree(x, given, 20)


def test_flat_and_peaked_rows():
    n = 50257
    x = np.zeros((3, n), dtype=np.float32)
    x[1, 7] = 30.0
    x[2] = -1e30
    x[2, 9] = 1e30
    logp, h, ids, logps = run(x, np.array([[5], [7], [9]]), 2)
    assert abs(h[0] - np.log(n)) < 1e-5 and h[1] >= 0 and h[2] == 0
    assert abs(logp[0, 0] + np.log(n)) < 1e-5 and logp[1, 0] <= 0 and logp[2, 0] == 0
    assert ids[1, 0] == 7 and ids[2, 0] == 9 and list(ids[0]) == [0, 1]


@pytest.mark.parametrize("size", [1.0, 1e3, 1.04e6, 1.05e6, 1e7, 1e30, 3.4028234e38])
def test_logits_of_any_size(size):
    """the two ways a thread's sums are taken (past 2^20 against the largest logit itself), a row that crosses from one to the
    other on the way, rows of the type's lowest value"""
    rng = np.random.default_rng(8)
    x = (rng.standard_normal((5, 20011)) * 2).astype(np.float32)
    x[0] += np.float32(size)
    x[1] -= np.float32(size)
    x[2, 10000:] += np.float32(size)
    x[3] = -np.float32(size)
    x[4, :3] = -np.float32(size)
    agree(x, rng.integers(0, 20011, (5, 3)), 9)


def test_rows_without_probabilities():
    """a NaN, an infinity, nothing but minus infinity: NaN and -1 in that row, the others as without it"""
    rng = np.random.default_rng(4)
    x = (rng.standard_normal((5, 9000))).astype(np.float32)
    given = rng.integers(0, 9000, (5, 1))
    clean = run(x, given, 3)
    x[1, 8999], x[2, 17], x[3] = np.nan, np.inf, -np.inf
    dirty = run(x, given, 3)
    for got, want in zip(dirty, clean):
        np.testing.assert_array_equal(got[[0, 4]], want[[0, 4]])
    for i in (1, 2, 3):
        assert np.isnan(dirty[0][i]).all() and np.isnan(dirty[1][i]) and (dirty[2][i] == -1).all()
        assert np.isnan(dirty[3][i]).all()


def test_tokens_outside_the_vocabulary():
    x = np.zeros((2, 100), dtype=np.float32)
    logp = run(x, np.array([[-1, 99], [100, 0]]), 0)[0]
    assert np.isnan(logp[0, 0]) and np.isnan(logp[1, 0])
    np.testing.assert_allclose([logp[0, 1], logp[1, 1]], -np.log(100), rtol=1e-6)


def test_parts_that_are_not_asked_for():
    rng = np.random.default_rng(5)
    x = rng.standard_normal((3, 700)).astype(np.float32)
    agree(x, None, 4, entropy=False)
    agree(x, rng.integers(0, 700, (3, 64)), 0)


def test_captured_calls_replay():
    lib, h = package().library(), hip()
    rng = np.random.default_rng(6)
    for m, n, top in ((1, 128256, 20), (64, 4099, 5)):
        xd, given = Dev((m, n), np.float32), rng.integers(0, n, (m, 1)).astype(np.int32)
        gd, logp, ent = upload(given), Dev((m, 1), np.float32), Dev(m, np.float32)
        ids, logps = Dev((m, top), np.int32), Dev((m, top), np.float32)
        need = lib.hk_logprobs_workspace(m, n, top)
        space = Dev(max(1, need), np.uint8, np.full(max(1, need), 0xFF))
        stream, graph, replay = ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_void_p()
        hip_check(h.hipStreamCreate(ctypes.byref(stream)))
        hip_check(h.hipStreamBeginCapture(stream, 2))
        check(lib.hk_logprobs(logp.ptr, ent.ptr, ids.ptr, logps.ptr, xd.ptr, n, gd.ptr, 1, m, n, top, space.ptr, need, stream))
        hip_check(h.hipStreamEndCapture(stream, ctypes.byref(graph)))
        hip_check(h.hipGraphInstantiate(ctypes.byref(replay), graph, None, None, 0))
        for _ in range(3):
            x = (rng.standard_normal((m, n)) * 3).astype(np.float32)
            hip_check(h.hipMemcpy(xd.ptr, ctypes.c_void_p(x.ctypes.data), xd.nbytes, 1))
            hip_check(h.hipGraphLaunch(replay, stream))
            hip_check(h.hipStreamSynchronize(stream))
            want = run(x, given, top)
            for got, w in zip((logp, ent, ids, logps), want):
                np.testing.assert_array_equal(got.numpy(), w)
            wl, wh, wi, wp = expected(x, given, top)
            np.testing.assert_array_equal(ids.numpy(), wi)
            np.testing.assert_allclose(logp.numpy(), wl, atol=1e-5, rtol=0)
        hip_check(h.hipGraphExecDestroy(replay))
        hip_check(h.hipGraphDestroy(graph))
        hip_check(h.hipStreamDestroy(stream))


@pytest.mark.parametrize("m, n", [(1500, 64), (100, 9000), (640, 4100)])
def test_probabilities_and_entropies_have_their_sign(m, n):
    """peaked rows: no probability above 1, no entropy below 0, whatever the largest logit rounds to"""
    rng = np.random.default_rng(n)
    x = np.empty((m, n), dtype=np.float32)
    top = rng.uniform(-40, 40, m).astype(np.float32)
    x[:] = top[:, None] - np.where(np.arange(m) % 2, 200.0, 25.0)[:, None]
    at = rng.integers(0, n, m)
    x[np.arange(m), at] = top
    logp, h, ids, logps = run(x, at[:, None], 5)
    assert (logp <= 0).all() and (logps <= 0).all() and (h >= 0).all()
    # rows of one token: its term is 2^t, t from -1 to 0, times 2^-t, two exponentials within 2^-23 of themselves and a product
    # rounded to 2^-24: Z within 2^-21 of 1. H is 2^t t plus -t Z, their roundings 2^-24 each and Z's error: with log Z 2^-20
    assert (logp[1::2] >= -2.0 ** -21).all() and (h[1::2] <= 2.0 ** -20).all()
    agree(x, at[:, None], 5)
