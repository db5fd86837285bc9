"""hk_cache_append / read / rewind / attention against the NumPy oracle: the cache's bytes exactly, the attention within the
derived bound of its float64 form."""
import ctypes

import numpy as np
import pytest

from cache_lib import BLOCK, RECENT, Cache, Model, rows
from gpu_lib import Dev, check, hip, hip_check, upload
from paths import package

pytestmark = pytest.mark.gpu

# query heads, kv heads, head size: every head size, groups of one to 32, odd ones
HEADS = [(4, 2, 16), (10, 5, 32), (6, 6, 48), (8, 8, 64), (12, 4, 96), (8, 2, 128), (7, 1, 128), (4, 2, 256), (32, 1, 64),
         (9, 1, 32), (3, 1, 16)]


def same_blocks(cache, model, end):
    q, s = cache.blocks()
    n = end // BLOCK
    np.testing.assert_array_equal(s[:, :n].view(np.uint32), model.s[:, :n].view(np.uint32))
    np.testing.assert_array_equal(q[:, :n], model.q[:, :n])


def within(got, model, q, pos, nh):
    want, off = model.attention(q, pos, nh)
    assert np.isfinite(got).all()
    worst = np.max(np.abs(got - want) / off)
    assert worst <= 1.0, worst
    return want


@pytest.mark.parametrize("hs, nkv", [(16, 3), (32, 1), (48, 6), (64, 2), (96, 4), (128, 8), (256, 2)])
@pytest.mark.parametrize("counts", [(1,), (31, 1, 1), (32,), (33, 31), (5, 150, 3, 200), (64, 96, 1), (7, 121), (7, 122, 1)])
def test_append_gives_the_exact_bytes_and_leaves_the_rest(hs, nkv, counts):
    rng = np.random.default_rng(hs + sum(counts))
    seq = 400
    cache, model, pos = Cache(nkv, hs, seq, fill=77), Model(nkv, hs, seq), 0
    for n in counts:
        k, v = rows(rng, n, nkv, hs)
        cache.append(k, v, pos)
        model.append(k, v, pos)
        pos += n
        same_blocks(cache, model, pos)
        # the latest positions in float32
        for w, name in enumerate(("recent_keys", "recent_values")):
            kept = cache.dev[name].numpy()
            for p in range(max(0, pos - RECENT), pos):
                np.testing.assert_array_equal(kept[p % RECENT], model.rows[w, p])
        np.testing.assert_array_equal(cache.read(0, pos, pos), model.read(0, pos, pos).astype(np.float32))
    q, s = cache.blocks()
    assert (q[0, pos // BLOCK:] == 77).all() and (q[1, pos // BLOCK:] == 77 - 128).all()
    assert (s[:, pos // BLOCK:] == np.float32(11)).all()


def test_quantization_at_its_borders():
    """ties to even and the values next to them, blocks of zeros, denormals and huge values"""
    nkv, hs = 4, 16
    rng = np.random.default_rng(3)
    n = 32 * 6
    k, v = np.zeros((n, nkv, hs), dtype=np.float32), np.zeros((n, nkv, hs), dtype=np.float32)
    for b in range(6):
        for h in range(nkv):
            for x in (k, v):
                largest = np.float32(rng.choice([127.0, 0.37, 2.0 ** -120, 1e-39, 1e38, 3.7e-9]))
                s = largest * np.float32(1 / 127)
                steps = rng.integers(-126, 126, (32, hs)) + 0.5
                near = (steps * np.float64(s)).astype(np.float32)
                for other in (np.nextafter(near, np.float32(1e38)), np.nextafter(near, np.float32(-1e38))):
                    near = np.where(rng.random(near.shape) < 0.3, other, near)
                near = np.clip(near, -largest, largest)
                near[0, 0] = largest
                x[b * 32:b * 32 + 32, h] = near
    k[64:96, 1] = 0
    cache, model = Cache(nkv, hs, n), Model(nkv, hs, n)
    cache.append(k.reshape(n, -1), v.reshape(n, -1), 0)
    model.append(k, v, 0)
    model.q = np.clip(model.q, -127, 127)
    same_blocks(cache, model, n)


@pytest.mark.parametrize("nh, nkv, hs", HEADS)
@pytest.mark.parametrize("pos, count", [(0, 1), (31, 1), (32, 1), (33, 1), (0, 33), (20, 50), (97, 1), (200, 3), (5, 160),
                                        (470, 7), (1027, 1)])
def test_attention(nh, nkv, hs, pos, count):
    rng = np.random.default_rng(pos * 7 + count + hs + nh)
    seq = pos + count
    cache, model = Cache(nkv, hs, seq, fill=91), Model(nkv, hs, seq)
    k, v = rows(rng, seq, nkv, hs)
    if pos:
        cache.append(k[:pos], v[:pos], 0)
        model.append(k[:pos], v[:pos], 0)
    cache.append(k[pos:], v[pos:], pos)
    model.append(k[pos:], v[pos:], pos)
    q = (rng.standard_normal((count, nh * hs)) * 1.5).astype(np.float32)
    within(cache.attention(q, k[pos:], v[pos:], pos, nh, pad=4 * (count % 3)), model, q, pos, nh)


@pytest.mark.parametrize("nh, nkv, hs", [(8, 2, 128), (6, 6, 48), (28, 4, 128), (4, 2, 256)])
@pytest.mark.parametrize("pos", [4095, 5003, 9000])
def test_attention_of_one_token_over_a_long_context(nh, nkv, hs, pos):
    rng = np.random.default_rng(pos + hs)
    cache, model = Cache(nkv, hs, pos + 1), Model(nkv, hs, pos + 1)
    k, v = rows(rng, pos + 1, nkv, hs)
    cache.append(k, v, 0)
    model.append(k, v, 0)
    # (the call's own row is the last one: the cache's recent rows hold the others of its block)
    q = (rng.standard_normal((1, nh * hs)) * 2).astype(np.float32)
    within(cache.attention(q, k[pos:], v[pos:], pos, nh), model, q, pos, nh)


@pytest.mark.parametrize("pos, count", [(1500, 37), (640, 300), (3, 700)])
def test_attention_of_a_prompt_behind_a_context(pos, count):
    nh, nkv, hs = 8, 2, 128
    rng = np.random.default_rng(count)
    cache, model = Cache(nkv, hs, pos + count), Model(nkv, hs, pos + count)
    k, v = rows(rng, pos + count, nkv, hs)
    for a, b in ((0, pos), (pos, pos + count)):
        cache.append(k[a:b], v[a:b], a)
        model.append(k[a:b], v[a:b], a)
    q = (rng.standard_normal((count, nh * hs))).astype(np.float32)
    within(cache.attention(q, k[pos:], v[pos:], pos, nh), model, q, pos, nh)


def test_scores_and_scales_far_apart():
    """a row's largest score growing block by block, one block's values a million times the others', values of zero, keys
    of zero: the running references follow"""
    nh, nkv, hs, n = 4, 1, 64, 32 * 12 + 5
    rng = np.random.default_rng(8)
    k, v = rows(rng, n, nkv, hs)
    k *= np.linspace(0.01, 4, n, dtype=np.float32)[:, None]
    v[64:96] *= 1e6
    v[128:160] *= 1e-6
    v[160:192] = 0
    k[192:224] = 0
    for order in (slice(None), slice(None, None, -1)):
        kk, vv = np.ascontiguousarray(k[order]), np.ascontiguousarray(v[order])
        cache, model = Cache(nkv, hs, n), Model(nkv, hs, n)
        cache.append(kk, vv, 0)
        model.append(kk, vv, 0)
        for scale in (0.01, 1.0, 6.0):
            q = (rng.standard_normal((n, nh * hs)) * scale).astype(np.float32)
            within(cache.attention(q, kk, vv, 0, nh), model, q, 0, nh)


def test_small_values_beside_a_block_of_large_ones_keep_their_bits():
    """a row whose probability lies on blocks of small values, behind a block of large values that it gives none: its error
    is measured against the small ones"""
    nh, nkv, hs, n = 2, 1, 32, 97
    rng = np.random.default_rng(4)
    k, v = rows(rng, n, nkv, hs, wide=0)
    k[:32, 0], k[32:, 0] = -40, 40
    v[:32] *= 1e8
    q = np.zeros((1, nh * hs), dtype=np.float32)
    q[0, ::hs] = 10.0
    cache, model = Cache(nkv, hs, n), Model(nkv, hs, n)
    cache.append(k, v, 0)
    model.append(k, v, 0)
    got = cache.attention(q, k[96:], v[96:], 96, nh)
    want, _ = model.attention(q, 96, nh)
    # the scores of the last 65 positions differ by what keys' 8 bits make of 40: about 1; those of the first lie 140 below.
    # A score of 70 is off by 2^-21 * 70 at most (its float32 steps), a probability by twice that: 7e-5 of the small values
    assert np.max(np.abs(got - want)) <= 2 * 2.0 ** -21 * 80 * np.abs(v[32:]).max()


@pytest.mark.parametrize("counts", [(150,), (1,) * 150, (37, 1, 95, 17), (96, 54)])
def test_a_token_is_the_same_however_the_tokens_before_it_were_split(counts):
    nh, nkv, hs, n = 8, 2, 64, 150
    rng = np.random.default_rng(5)
    k, v = rows(rng, n, nkv, hs)
    q = rng.standard_normal((n, nh * hs)).astype(np.float32)
    cache, model = Cache(nkv, hs, n), Model(nkv, hs, n)
    model.append(k, v, 0)
    pos, got = 0, []
    for c in counts:
        cache.append(k[pos:pos + c], v[pos:pos + c], pos)
        got.append(cache.attention(q[pos:pos + c], k[pos:pos + c], v[pos:pos + c], pos, nh))
        pos += c
    same_blocks(cache, model, n)
    within(np.concatenate(got), model, q, 0, nh)


def test_tokens_taken_again():
    """a step back within the latest positions gives the bytes of the tokens that are taken; further back, after
    hk_cache_rewind, the block's earlier rows stand as their 8-bit values"""
    nkv, hs, seq = 2, 64, 600
    rng = np.random.default_rng(6)
    cache, model = Cache(nkv, hs, seq), Model(nkv, hs, seq)
    k, v = rows(rng, 300, nkv, hs)
    cache.append(k, v, 0)
    model.append(k, v, 0)
    back = 300 - (RECENT - BLOCK)
    k, v = rows(rng, 77, nkv, hs)
    cache.append(k, v, back)
    model.append(k, v, back)
    same_blocks(cache, model, back + 77)
    cache.rewind(50)
    model.rewind(50)
    k, v = rows(rng, 30, nkv, hs)
    cache.append(k, v, 50)
    model.append(k, v, 50)
    same_blocks(cache, model, 80)
    q = rng.standard_normal((30, 4 * hs)).astype(np.float32)
    within(cache.attention(q, k, v, 50, 4), model, q, 50, 4)


@pytest.mark.parametrize("what", ["query", "key", "value", "infinite value"])
def test_what_is_not_finite_reaches_only_the_rows_that_see_it(what):
    nh, nkv, hs, n, at = 4, 2, 64, 100, 41
    rng = np.random.default_rng(7)
    k, v = rows(rng, n, nkv, hs)
    q = rng.standard_normal((n, nh * hs)).astype(np.float32)
    clean, dirty = Cache(nkv, hs, n), Cache(nkv, hs, n)
    clean.append(k, v, 0)
    want = clean.attention(q, k, v, 0, nh)
    if what == "query":
        q[at, 5] = np.inf
    elif what == "key":
        k[at, hs + 3] = np.nan
    else:
        v[at, hs + 3] = np.nan if what == "value" else -np.inf
    dirty.append(k, v, 0)
    got = dirty.attention(q, k, v, 0, nh)
    if what == "query":
        assert np.isnan(got[at, 0]).all()
        got[at, 0] = want[at, 0]
    else:  # kv head 1: query heads 2 and 3, from the token on
        assert np.isnan(got[at:, 2:]).any(-1).all()
        got[at:, 2:] = want[at:, 2:]
    np.testing.assert_array_equal(got, want)


def test_rows_behind_the_tokens_do_not_matter():
    """what lies behind the last position (an earlier, longer use of the same buffers) is not read"""
    nh, nkv, hs, n = 8, 2, 128, 77
    rng = np.random.default_rng(9)
    k, v = rows(rng, n, nkv, hs)
    q = rng.standard_normal((n, nh * hs)).astype(np.float32)
    fresh, used = Cache(nkv, hs, 400), Cache(nkv, hs, 400)
    k2, v2 = rows(rng, 400, nkv, hs)
    k2[:], v2[:] = np.nan, np.inf
    used.append(k2, v2, 0)
    got = []
    for cache in (fresh, used):
        cache.append(k, v, 0)
        got.append(cache.attention(q, k, v, 0, nh))
        got.append(cache.attention(q[76:], k[76:], v[76:], 76, nh))
    assert np.isfinite(got[2]).all() and np.isfinite(got[3]).all()
    np.testing.assert_array_equal(got[0], got[2])
    np.testing.assert_array_equal(got[1], got[3])


@pytest.mark.parametrize("pos, count", [(300, 1), (301, 1), (0, 90), (40, 12)])
def test_captured_calls_replay(pos, count):
    """append and attention captured on a stream and replayed with other inputs between the replays"""
    nh, nkv, hs, seq = 8, 2, 128, 512
    rng = np.random.default_rng(pos)
    lib = package().library()
    cache, model = Cache(nkv, hs, seq), Model(nkv, hs, seq)
    k, v = rows(rng, pos + count, nkv, hs)
    if pos:
        cache.append(k[:pos], v[:pos], 0)
        model.append(k[:pos], v[:pos], 0)
    bufs = {n: Dev((count, w * hs), np.float32) for n, w in (("q", nh), ("k", nkv), ("v", nkv), ("out", nh))}
    need = lib.hk_cache_workspace(cache.ref, nh, count)
    space = Dev(max(1, need), np.uint8)
    h = hip()
    stream, graph, run = ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_void_p()
    hip_check(h.hipStreamCreate(ctypes.byref(stream)))
    hip_check(h.hipStreamBeginCapture(stream, 2))
    check(lib.hk_cache_append(cache.ref, bufs["k"].ptr, bufs["v"].ptr, nkv * hs, count, pos, stream))
    check(lib.hk_cache_attention(bufs["out"].ptr, bufs["q"].ptr, bufs["k"].ptr, bufs["v"].ptr, cache.ref, nh, nh * hs,
                                 nkv * hs, nh * hs, count, pos, space.ptr, need, stream))
    hip_check(h.hipStreamEndCapture(stream, ctypes.byref(graph)))
    hip_check(h.hipGraphInstantiate(ctypes.byref(run), graph, None, None, 0))
    for _ in range(3):
        q = rng.standard_normal((count, nh * hs)).astype(np.float32)
        kk, vv = rows(rng, count, nkv, hs)
        for name, x in (("q", q), ("k", kk), ("v", vv)):
            x = np.ascontiguousarray(x)
            hip_check(h.hipMemcpy(bufs[name].ptr, ctypes.c_void_p(x.ctypes.data), bufs[name].nbytes, 1))
        hip_check(h.hipGraphLaunch(run, stream))
        hip_check(h.hipStreamSynchronize(stream))
        model.append(kk, vv, pos)
        got = bufs["out"].numpy().reshape(count, nh, hs)
        within(got, model, q, pos, nh)
        same_blocks(cache, model, pos + count)
        np.testing.assert_array_equal(got, cache.attention(q, kk, vv, pos, nh))  # an eager call between the replays
    hip_check(h.hipGraphExecDestroy(run))
    hip_check(h.hipGraphDestroy(graph))
    hip_check(h.hipStreamDestroy(stream))


def test_two_streams_at_once():
    """two caches on two streams, each with its own workspace: the results of the calls one after the other"""
    nh, nkv, hs, n = 8, 2, 128, 2100
    lib, h = package().library(), hip()
    rng = np.random.default_rng(11)
    work = []
    for _ in range(2):
        cache = Cache(nkv, hs, n)
        k, v = rows(rng, n, nkv, hs)
        cache.append(k, v, 0)
        q = rng.standard_normal((1, nh * hs)).astype(np.float32)
        want = cache.attention(q, k[-1:], v[-1:], n - 1, nh)
        need = lib.hk_cache_workspace(cache.ref, nh, 1)
        stream = ctypes.c_void_p()
        hip_check(h.hipStreamCreate(ctypes.byref(stream)))
        work.append((cache, stream, upload(q), upload(k[-1:]), upload(v[-1:]), Dev((1, nh * hs), np.float32),
                     Dev(max(1, need), np.uint8), need, want))
    for _ in range(20):
        for cache, stream, q, k, v, out, space, need, _ in work:
            check(lib.hk_cache_attention(out.ptr, q.ptr, k.ptr, v.ptr, cache.ref, nh, nh * hs, nkv * hs, nh * hs, 1,
                                         n - 1, space.ptr, need, stream))
    for cache, stream, q, k, v, out, space, need, want in work:
        hip_check(h.hipStreamSynchronize(stream))
        np.testing.assert_array_equal(out.numpy().reshape(want.shape), want)
        hip_check(h.hipStreamDestroy(stream))


def test_offsets_past_32_bits():
    """a cache whose keys alone pass 2^32 bytes: positions near its end are read where they were written"""
    nh, nkv, hs = 16, 16, 256
    seq = (1 << 32) // (nkv * hs) + 4096
    cache = Cache.__new__(Cache)
    pk = package()
    cache.nkv, cache.hs, cache.seq_len, cache.dev = nkv, hs, seq, {}
    for name, (shape, dtype) in pk.cache_shapes(nkv, hs, seq).items():
        d = Dev.__new__(Dev)
        d.shape, d.dtype = shape, np.dtype(dtype)
        d.nbytes, d.ptr = int(np.prod(shape)) * d.dtype.itemsize, ctypes.c_void_p()
        hip_check(hip().hipMalloc(ctypes.byref(d.ptr), d.nbytes))
        cache.dev[name] = d
    cache.c = pk.HkCache(n_kv_heads=nkv, head_size=hs, seq_len=seq, **{k: d.ptr.value for k, d in cache.dev.items()})
    cache.ref = ctypes.byref(cache.c)
    rng = np.random.default_rng(12)
    start = seq // BLOCK * BLOCK - 4 * BLOCK
    k, v = rows(rng, 3 * BLOCK, nkv, hs)
    cache.append(k, v, start)
    model = Model(nkv, hs, 3 * BLOCK)
    model.append(k, v, 0)
    end = start + 3 * BLOCK
    np.testing.assert_array_equal(cache.read(start, 3 * BLOCK, end), model.read(0, 3 * BLOCK, 3 * BLOCK).astype(np.float32))


def test_a_conversation_with_its_probabilities():
    """the operators as a program runs them: a prompt, then steps of one token over the cache; the attention's rows as
    logits, the most probable token's probability taken from them"""
    nh, nkv, hs, n = 8, 2, 64, 70
    rng = np.random.default_rng(13)
    lib = package().library()
    cache, model = Cache(nkv, hs, 200), Model(nkv, hs, 200)
    k, v = rows(rng, n, nkv, hs)
    q = rng.standard_normal((n, nh * hs)).astype(np.float32)
    pos = 0
    for c in (60,) + (1,) * 10:
        cache.append(k[pos:pos + c], v[pos:pos + c], pos)
        model.append(k[pos:pos + c], v[pos:pos + c], pos)
        out = cache.attention(q[pos:pos + c], k[pos:pos + c], v[pos:pos + c], pos, nh)
        want = within(out, model, q[pos:pos + c], pos, nh)
        logits = upload(out.reshape(c, nh * hs))
        need = lib.hk_logprobs_workspace(c, nh * hs, 1)
        ids, logps, space = Dev((c, 1), np.int32), Dev((c, 1), np.float32), Dev(max(1, need), np.uint8)
        check(lib.hk_logprobs(None, None, ids.ptr, logps.ptr, logits.ptr, nh * hs, None, 0, c, nh * hs, 1, space.ptr,
                              need, None))
        x = want.reshape(c, -1)
        lse = np.log(np.exp(x - x.max(-1, keepdims=True)).sum(-1)) + x.max(-1)
        np.testing.assert_array_equal(ids.numpy()[:, 0], out.reshape(c, -1).argmax(-1))
        np.testing.assert_allclose(logps.numpy()[:, 0], x.max(-1) - lse, atol=1e-4, rtol=0)  # (the bound of `within`)
        pos += c


@pytest.mark.parametrize("nh, nkv, hs", [(200, 200, 16), (400, 200, 32)])
@pytest.mark.parametrize("pos, count", [(700, 1), (690, 2), (500, 9)])
def test_attention_of_few_tokens_with_many_kv_heads(nh, nkv, hs, pos, count):
    """as many tiles as waves fill the card with, from one token on"""
    rng = np.random.default_rng(pos + nh)
    cache, model = Cache(nkv, hs, pos + count), Model(nkv, hs, pos + count)
    k, v = rows(rng, pos + count, nkv, hs)
    cache.append(k, v, 0)
    model.append(k, v, 0)
    q = rng.standard_normal((count, nh * hs)).astype(np.float32)
    within(cache.attention(q, k[pos:], v[pos:], pos, nh), model, q, pos, nh)


@pytest.mark.parametrize("nh, nkv, hs", [(22, 2, 64), (8, 8, 128), (32, 1, 16), (10, 5, 32), (4, 2, 256), (200, 200, 16)])
@pytest.mark.parametrize("pos, count", [(0, 1), (5003, 1), (5001, 6), (4999, 37), (90, 300), (3000, 1000)])
def test_nothing_is_written_behind_the_workspace(nh, nkv, hs, pos, count):
    lib, seq = package().library(), pos + count
    cache = Cache(nkv, hs, seq)
    q, k = Dev((count, nh * hs), np.float32), Dev((count, nkv * hs), np.float32)
    out = Dev((count, nh * hs), np.float32)
    need = lib.hk_cache_workspace(cache.ref, nh, count)
    assert need >= 0
    space = Dev(need + 65536, np.uint8, np.full(need + 65536, 0xA5))
    check(lib.hk_cache_attention(out.ptr, q.ptr, k.ptr, k.ptr, cache.ref, nh, nh * hs, nkv * hs, nh * hs, count, pos,
                                 space.ptr, need, None))
    assert (space.numpy()[need:] == 0xA5).all()


@pytest.mark.parametrize("sign", [1, -1])
def test_an_infinite_key_reaches_every_row_that_sees_it(sign):
    """also those whose score it takes to minus infinity: in its own block, and once that is in 8 bits"""
    nh, nkv, hs, n, at = 4, 2, 64, 100, 41
    rng = np.random.default_rng(17)
    k, v = rows(rng, n, nkv, hs)
    q = rng.standard_normal((n, nh * hs)).astype(np.float32)
    k[at, hs + 3] = sign * np.inf
    cache = Cache(nkv, hs, n)
    cache.append(k, v, 0)
    got = cache.attention(q, k, v, 0, nh)
    assert np.isnan(got[at:, 2:]).any(-1).all()
    assert np.isfinite(got[:at]).all() and np.isfinite(got[:, :2]).all()
    few = Cache(nkv, hs, n)
    few.append(k[:50], v[:50], 0)
    for p in (40, 41, 49):
        one = few.attention(q[p:p + 1], k[p:p + 1], v[p:p + 1], p, nh)
        assert np.isfinite(one[0, :2]).all() and np.isnan(one[0, 2:]).any(-1).all() == (p >= at)


@pytest.mark.parametrize("nh, nkv, hs, pos, count", [(6, 6, 48, 40, 1), (8, 2, 128, 700, 1), (8, 2, 128, 20, 50), (4, 2, 256, 70, 40),
                                                     (48, 48, 16, 20, 200), (96, 48, 64, 33, 170)])
@pytest.mark.parametrize("size", [1e-35, 1e-30, 3e19, 1e35, 1e38])
@pytest.mark.parametrize("which", ["all", "the last", "one in three"])
def test_values_of_any_size(nh, nkv, hs, pos, count, size, which):
    """values up to 3.3e38 and down to 1e-35, in the token's own block as behind it: the attention lies between them, and a row
    that sees no large one keeps the bits of its small ones"""
    rng = np.random.default_rng(count + hs)
    n = pos + count
    cache, model = Cache(nkv, hs, n), Model(nkv, hs, n)
    k, v = rows(rng, n, nkv, hs)
    large = np.zeros(n, dtype=bool)
    large[slice(None) if which == "all" else slice(n - 1, None) if which == "the last" else slice(1, None, 3)] = True
    v[large] = np.clip(v[large], -3.3, 3.3) * np.float32(size)
    for a, b in ((0, pos), (pos, n)):
        cache.append(k[a:b], v[a:b], a)
        model.append(k[a:b], v[a:b], a)
    q = rng.standard_normal((count, nh * hs)).astype(np.float32)
    got = cache.attention(q, k[pos:], v[pos:], pos, nh)
    for i in sorted({0, count // 3, count // 2, count - 2, count - 1} & set(range(count))):
        within(got[i:i + 1], model, q[i:i + 1], pos + i, nh)


@pytest.mark.parametrize("nh, nkv, hs", [(31, 1, 128), (62, 2, 128), (15, 1, 256), (32, 1, 96)])
@pytest.mark.parametrize("pos, count", [(700, 1), (690, 5)])
def test_groups_whose_outputs_fill_the_workgroups_memory(nh, nkv, hs, pos, count):
    rng = np.random.default_rng(nh)
    cache, model = Cache(nkv, hs, pos + count), Model(nkv, hs, pos + count)
    k, v = rows(rng, pos + count, nkv, hs)
    cache.append(k, v, 0)
    model.append(k, v, 0)
    q = rng.standard_normal((count, nh * hs)).astype(np.float32)
    within(cache.attention(q, k[pos:], v[pos:], pos, nh), model, q, pos, nh)


@pytest.mark.parametrize("seed", range(6))
def test_steps_back_one_after_the_other(seed):
    """steps back by the rule hk_cache_append states: the float32 rows that are held lie behind the furthest position
    written, not behind the last call's end; anywhere else goes through hk_cache_rewind. The first sequence: 300 positions,
    one token at 204, then back to 120"""
    nh, nkv, hs, seq = 4, 2, 32, 700
    rng = np.random.default_rng(seed)
    cache, model = Cache(nkv, hs, seq), Model(nkv, hs, seq)
    start = furthest = end = whole = 0
    for step in range(12):
        if seed == 0 and step < 3:
            pos, count = ((0, 300), (204, 1), (120, 50))[step]
        else:
            back = [0, int(rng.integers(0, 97)), int(rng.integers(0, end + 1))][int(rng.integers(0, 3))]
            pos = max(0, end - back)
            count = min(int(rng.choice([1, 2, 30, 100, 200])), seq - pos)
            if count < 1:
                pos, count = 450, 1
        first = pos // BLOCK * BLOCK
        if not (max(start, furthest - RECENT) <= first and pos <= furthest):
            if pos % BLOCK:
                cache.rewind(pos)
                model.rewind(pos)
            start, furthest = first, pos
        k, v = rows(rng, count, nkv, hs)
        cache.append(k, v, pos)
        model.append(k, v, pos)
        end = pos + count
        furthest, whole = max(furthest, end), max(whole, end)
        same_blocks(cache, model, whole)
        q = rng.standard_normal((count, nh * hs)).astype(np.float32)
        got = cache.attention(q, k, v, pos, nh)
        for i in {0, count - 1}:
            within(got[i:i + 1], model, q[i:i + 1], pos + i, nh)
        np.testing.assert_array_equal(cache.read(0, end, end), model.read(0, end, end).astype(np.float32))
