"""hk_cache_attention where a call has many tiles of rows or a long context behind it, every token against the float64 form."""
import ctypes

import numpy as np
import pytest

from cache_lib import BLOCK, Cache, Model, rows
from gpu_lib import Dev, check, hip, hip_check, upload
from paths import package

pytestmark = pytest.mark.gpu


def attention64(model, q, pos, nh):
    """Model.attention's result and bound, a head's tokens at once"""
    count, hs, nkv = len(q), model.hs, model.nkv
    group, end, lo = nh // nkv, pos + count, pos // BLOCK * BLOCK
    old = (end - 1) // BLOCK
    k8, v8 = ((model.q[w, :old] * model.s[w, :old].astype(np.float64)[:, :, None, None]) for w in range(2))
    at = np.arange(pos, end)
    first = (at // BLOCK * BLOCK)[:, None]
    j = np.concatenate([np.arange(old * BLOCK), np.arange(lo, end)])
    eight = np.arange(len(j)) < old * BLOCK
    seen = np.where(eight[None], j[None] < first, (j[None] >= first) & (j[None] <= at[:, None]))
    q = q.astype(np.float64).reshape(count, nh, hs)
    out, off = np.zeros((count, nh, hs)), np.zeros((count, nh, 1))
    for g in range(nkv):
        k, v = (np.concatenate([x[:, g].reshape(-1, hs), model.rows[w, lo:end, g].astype(np.float64)])
                for w, x in ((0, k8), (1, v8)))
        largest_k = np.where(seen, np.abs(k).sum(-1)[None], 0).max(-1)
        largest_v = np.where(seen, np.abs(v).max(-1)[None], 0).max(-1)
        for h in range(g * group, (g + 1) * group):
            s = q[:, h] @ k.T / np.sqrt(hs)
            largest_s = np.where(seen, np.abs(s), 0).max(-1)
            s[~seen] = -np.inf
            e = np.exp(s - s.max(-1, keepdims=True))
            out[:, h] = e @ v / e.sum(-1, keepdims=True)
            ds = 2.0 ** -22 * np.abs(q[:, h]).max(-1) * largest_k / np.sqrt(hs) + 2.0 ** -21 * largest_s
            off[:, h, 0] = 3 * largest_v * (2 * ds + 2.0 ** -21 + (seen.sum(-1) / 16 + 32) * 2.0 ** -24)
    return out, off


def made(nh, nkv, hs, pos, count):
    """a cache and its model that hold pos + count positions, the last count as one call"""
    rng = np.random.default_rng(nh * hs + pos + count)
    n = pos + count
    cache, model = Cache(nkv, hs, n), Model(nkv, hs, n)
    k, v = rows(rng, n, nkv, hs)
    for a, b in ((0, pos), (pos, n)):
        if b > a:
            cache.append(k[a:b], v[a:b], a)
            model.append(k[a:b], v[a:b], a)
    return cache, model, k[pos:], v[pos:], rng.standard_normal((count, nh * hs)).astype(np.float32)


def within(cache, model, k, v, q, pos, nh, pad=0):
    got = cache.attention(q, k, v, pos, nh, pad)
    want, off = attention64(model, q, pos, nh)
    worst = (np.abs(got - want) / off).max((1, 2))
    assert np.isfinite(got).all() and worst.max() <= 1.0, (worst.max(), int(worst.argmax()))


# a prompt's tiles (of 32 rows, token and query head, of one kv head) one a wave: every head size; an odd and an even number of
# the rows of tiles that workgroups take from both ends, last rows that are not whole; the blocks in parts and not; groups whose
# rows do not fill a tile
PROMPTS = [(32, 32, 16, 0, 1100), (14, 14, 16, 37, 500), (20, 10, 32, 0, 333), (64, 32, 32, 5, 555), (12, 12, 48, 0, 600),
           (48, 48, 48, 333, 700), (8, 8, 64, 0, 800), (66, 66, 64, 20, 520), (12, 4, 96, 0, 400), (48, 16, 96, 7, 600),
           (32, 8, 128, 0, 1000), (32, 8, 128, 0, 1500), (28, 4, 128, 101, 700), (9, 3, 128, 31, 550), (16, 8, 256, 0, 500),
           (16, 8, 256, 37, 1100), (26, 13, 256, 64, 250), (7, 1, 128, 0, 1024), (32, 1, 64, 900, 200)]


@pytest.mark.parametrize("nh, nkv, hs, pos, count", PROMPTS)
def test_prompts_of_many_tiles(nh, nkv, hs, pos, count):
    cache, model, k, v, q = made(nh, nkv, hs, pos, count)
    within(cache, model, k, v, q, pos, nh, pad=4 * (count % 3))


@pytest.mark.parametrize("nh, nkv, hs, pos, count", [(64, 64, 16, 4001, 1), (32, 32, 32, 8003, 1), (64, 16, 48, 16100, 1),
                                                     (8, 8, 128, 33001, 1), (16, 8, 128, 32700, 5), (16, 8, 256, 33001, 1)])
def test_few_tokens_behind_a_context_that_takes_more_parts(nh, nkv, hs, pos, count):
    """contexts past which a tile's blocks go to two workgroups a CU (of 256 values they do not)"""
    cache, model, k, v, q = made(nh, nkv, hs, pos, count)
    within(cache, model, k, v, q, pos, nh)


@pytest.mark.parametrize("count", [1, 33, 420])
def test_attention_past_32_bits_of_bytes(count):
    """keys and values of 2^32 bytes and more: zeros but for the last blocks, whose scores lie far above theirs"""
    nh, nkv, hs = 16, 16, 256
    seq = (1 << 32) // (nkv * hs) + 4096
    cache = Cache.__new__(Cache)
    pk = package()
    cache.nkv, cache.hs, cache.seq_len, cache.dev = nkv, hs, seq, {}
    for name, (shape, dtype) in pk.cache_shapes(nkv, hs, seq).items():
        d = Dev.__new__(Dev)
        d.shape, d.dtype = shape, np.dtype(dtype)
        d.nbytes, d.ptr = int(np.prod(shape, dtype=np.int64)) * d.dtype.itemsize, ctypes.c_void_p()
        hip_check(hip().hipMalloc(ctypes.byref(d.ptr), ctypes.c_size_t(d.nbytes)))
        hip_check(hip().hipMemset(d.ptr, 0, ctypes.c_size_t(d.nbytes)))
        cache.dev[name] = d
    cache.c = pk.HkCache(n_kv_heads=nkv, head_size=hs, seq_len=seq, **{k: d.ptr.value for k, d in cache.dev.items()})
    cache.ref = ctypes.byref(cache.c)
    rng = np.random.default_rng(count)
    start, n = seq // BLOCK * BLOCK - 20 * BLOCK, 64 + count
    model = Model(nkv, hs, n)
    k, v = rows(rng, n, nkv, hs, wide=0)
    toward = rng.standard_normal((nkv, hs))
    k = (k.reshape(n, nkv, hs) * 0.25 + toward).astype(np.float32).reshape(n, -1)
    q = (rng.standard_normal((count, nh, hs)) * 0.25 + 3 * toward).astype(np.float32).reshape(count, -1)
    for a, b in ((0, 64), (64, n)):
        cache.append(k[a:b], v[a:b], start + a)
        model.append(k[a:b], v[a:b], a)
    got = cache.attention(q, k[64:], v[64:], start + 64, nh)
    want, off = attention64(model, q, 64, nh)
    # the positions before `start` have score 0 and value 0: where a row's largest score lies 20 above their number's logarithm
    # they weigh 2^-28 of it at most, nothing to the bound's 2^-20
    for i in range(count):
        s = np.einsum("hd,hd->h", q[i].reshape(nh, hs).astype(np.float64), k[64 + i].reshape(nkv, hs).astype(np.float64)) / 16
        assert s.min() > np.log(start) + 20
    assert (np.abs(got - want) <= off).all()


@pytest.mark.parametrize("nh, nkv, hs, count", [(12, 12, 48, 600), (16, 8, 256, 560), (32, 8, 128, 1030)])
@pytest.mark.parametrize("what", ["query", "key", "value", "infinite value", "infinite key"])
def test_what_is_not_finite_in_a_prompt_of_many_tiles(nh, nkv, hs, count, what):
    """it reaches the rows that see it and leaves the bits of the others"""
    cache, _, k, v, q = made(nh, nkv, hs, 0, count)
    want, at, group = cache.attention(q, k, v, 0, nh), 401, nh // nkv
    if what == "query":
        q[at, hs + 5] = np.nan
    else:
        (k if "key" in what else v)[at, hs + 3] = np.inf if "infinite" in what else np.nan
    dirty = Cache(nkv, hs, count)
    dirty.append(k, v, 0)
    got = dirty.attention(q, k, v, 0, nh)
    seen = np.zeros((count, nh), dtype=bool)
    if what == "query":
        seen[at, 1] = True
    else:
        seen[at:, group:2 * group] = True
    assert np.isnan(got[seen]).any(-1).all() and (what == "value" or "infinite value" == what or np.isnan(got[seen]).all())
    np.testing.assert_array_equal(got[~seen], want[~seen])


@pytest.mark.parametrize("nh, nkv, hs, count", [(12, 12, 48, 600), (16, 8, 256, 560), (32, 8, 128, 1030)])
def test_scores_and_scales_far_apart_in_a_prompt_of_many_tiles(nh, nkv, hs, count):
    rng = np.random.default_rng(hs)
    k, v = rows(rng, count, nkv, hs)
    k *= np.linspace(0.01, 4, count, dtype=np.float32)[:, None]
    v[64:96] *= 1e6
    v[128:160] *= 1e-6
    v[160:192] = 0
    k[192:224] = 0
    v[300:330] *= 1e30
    for order in (slice(None), slice(None, None, -1)):
        kk, vv = np.ascontiguousarray(k[order]), np.ascontiguousarray(v[order])
        cache, model = Cache(nkv, hs, count), Model(nkv, hs, count)
        cache.append(kk, vv, 0)
        model.append(kk, vv, 0)
        q = (rng.standard_normal((count, nh * hs)) * 2).astype(np.float32)
        within(cache, model, kk, vv, q, 0, nh)
