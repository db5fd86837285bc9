"""hk_cache_* and hk_logprobs refuse what they do not take, before anything touches the device (no GPU needed)."""
import ctypes

import pytest

from paths import package

GOOD = dict(keys=1 << 20, values=2 << 20, scales=3 << 20, recent_keys=4 << 20, recent_values=5 << 20, n_kv_heads=2,
            head_size=64, seq_len=1000)


def cache(**change):
    return package().HkCache(**{**GOOD, **change})


def append(c, k=1 << 21, v=1 << 22, stride=128, count=5, pos=7):
    return package().library().hk_cache_append(ctypes.byref(c) if c else None, k, v, stride, count, pos, None)


def attention(c, out=1 << 20, q=1 << 21, k=1 << 22, v=1 << 23, heads=8, q_stride=512, kv_stride=128, out_stride=512, count=1,
              pos=7, workspace=1 << 24, size=1 << 30):
    return package().library().hk_cache_attention(out, q, k, v, ctypes.byref(c), heads, q_stride, kv_stride, out_stride,
                                                  count, pos, workspace, size, None)


def refused(rc, code="HE_E_ARG", text=b""):
    pk = package()
    assert rc == getattr(pk.hip_engine, code)
    message = pk.library().he_last_error()
    assert message.startswith(b"hk_") and text in message, message


@pytest.mark.parametrize("change", [dict(head_size=80), dict(head_size=0), dict(n_kv_heads=0), dict(seq_len=0),
                                    dict(seq_len=(1 << 24) + 1), dict(keys=None), dict(values=None), dict(scales=None),
                                    dict(recent_keys=None), dict(recent_values=None), dict(keys=(1 << 20) + 4)])
def test_caches_that_are_refused(change):
    lib = package().library()
    c = cache(**change)
    refused(append(c))
    refused(attention(c))
    refused(lib.hk_cache_read(1 << 20, 1 << 21, ctypes.byref(c), 0, 4, 8, None))
    refused(lib.hk_cache_rewind(ctypes.byref(c), 5, None))


@pytest.mark.parametrize("change, code, text", [
    (dict(k=None), "HE_E_ARG", b"k or v"), (dict(v=None), "HE_E_ARG", b"k or v"),
    (dict(k=(1 << 21) + 8), "HE_E_ARG", b"16-byte"), (dict(stride=124), "HE_E_ARG", b"kv_stride"),
    (dict(stride=130), "HE_E_ARG", b"kv_stride"), (dict(count=0), "HE_E_ARG", b"count"),
    (dict(count=-1), "HE_E_ARG", b"count"), (dict(pos=-1), "HE_E_ARG", b"pos"),
    (dict(pos=996), "HE_E_STATE", b"seq_len"), (dict(pos=2147483647), "HE_E_STATE", b"seq_len"),
    (dict(count=2147483647), "HE_E_STATE", b"seq_len")])
def test_rows_that_are_refused(change, code, text):
    refused(append(cache(), **change), code, text)
    change = {"kv_stride" if name == "stride" else name: x for name, x in change.items()}
    refused(attention(cache(), **{"count": 5, **change}), code, text)


@pytest.mark.parametrize("change, text", [
    (dict(out=None), b"out or q"), (dict(q=None), b"out or q"), (dict(q=(1 << 21) + 4), b"16-byte"),
    (dict(heads=7), b"n_heads"), (dict(heads=0), b"n_heads"), (dict(heads=66), b"n_heads"), (dict(q_stride=508), b"q_stride"),
    (dict(out_stride=514), b"out_stride")])
def test_attention_calls_that_are_refused(change, text):
    refused(attention(cache(), **change), text=text)


def test_a_workspace_that_is_refused():
    lib, c = package().library(), cache(seq_len=100000)
    need = lib.hk_cache_workspace(ctypes.byref(c), 8, 1)
    assert need >= 0
    if need:
        for change in (dict(workspace=None), dict(size=need - 1), dict(workspace=(1 << 24) + 8)):
            refused(attention(c, **change), text=b"workspace")
    refused(lib.hk_cache_workspace(ctypes.byref(c), 7, 1))
    refused(lib.hk_cache_workspace(ctypes.byref(c), 8, 0))
    refused(lib.hk_cache_workspace(None, 8, 1))


def test_reads_and_rewinds_that_are_refused():
    lib, c = package().library(), cache()
    for start, count, end in ((-1, 2, 8), (0, -1, 8), (4, 5, 8), (0, 4, 1001), (2147483647, 2147483647, 1000)):
        refused(lib.hk_cache_read(1 << 20, 1 << 21, ctypes.byref(c), start, count, end, None), text=b"range")
    refused(lib.hk_cache_read(None, 1 << 21, ctypes.byref(c), 0, 4, 8, None), text=b"null")
    for pos in (-1, 1000):
        refused(lib.hk_cache_rewind(ctypes.byref(c), pos, None), text=b"context")
    refused(append(None), text=b"null")


@pytest.mark.parametrize("change, text", [
    (dict(m=0), b"m and n"), (dict(n=0), b"m and n"), (dict(top=33), b"top"), (dict(top=-1), b"top"),
    (dict(logits=None), b"logits"), (dict(logits=(1 << 20) + 2), b"logits"), (dict(stride=99), b"stride"),
    (dict(given=None), b"given"), (dict(logp=None), b"given"), (dict(n_given=-1), b"given"), (dict(ids=None), b"ids"),
    (dict(logps=None), b"ids"), (dict(n_given=0, top=0, entropy=None), b"nothing")])
def test_log_probabilities_that_are_refused(change, text):
    args = dict(logp=1 << 21, entropy=1 << 22, ids=1 << 23, logps=1 << 24, logits=1 << 20, stride=100, given=1 << 25,
                n_given=1, m=2, n=100, top=3, workspace=1 << 26, size=1 << 30)
    args.update(change)
    refused(package().library().hk_logprobs(*args.values(), None), text=text)


@pytest.mark.parametrize("change", [dict(keys=(1 << 20) + 4), dict(values=(1 << 21) + 8)])
def test_reads_into_rows_that_are_not_aligned(change):
    to = dict(keys=1 << 20, values=1 << 21)
    to.update(change)
    refused(package().library().hk_cache_read(to["keys"], to["values"], ctypes.byref(cache()), 0, 4, 8, None), text=b"16-byte")


@pytest.mark.parametrize("m, n", [((1 << 30) + 1, 1), (2147483647, 1), (1, (1 << 30) + 1), (2147483647, 2147483647)])
def test_more_rows_or_logits_than_are_counted(m, n):
    refused(package().library().hk_logprobs_workspace(m, n, 0), text=b"2^30")
    refused(package().library().hk_logprobs(1 << 21, 1 << 22, None, None, 1 << 20, n, 1 << 25, 1, m, n, 0, 1 << 26, 1 << 40, None),
            text=b"2^30")
