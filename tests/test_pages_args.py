"""hk_pages_* and hk_matmul_four refuse what they do not take, before anything touches the device (no GPU needed); and
quantize_four's bytes."""
import ctypes

import numpy as np
import pytest

from paths import package

GOOD = dict(keys=1 << 20, values=2 << 20, tables=3 << 20, refs=4 << 20, n_layers=2, n_pages=100, n_kv_heads=2, page_size=64,
            head_size=64, half=1, n_seqs=10, table_size=20)


def made(**change):
    return package().HkPages(**{**GOOD, **change})


def calls(c):
    lib, ref = package().library(), ctypes.byref(c) if c else None
    a, s = 1 << 21, 1 << 24
    return [lambda: lib.hk_pages_fork(ref, a, a, a, 3, a, None),
            lambda: lib.hk_pages_reserve(ref, a, a, a, 3, a, s, 1 << 40, None),
            lambda: lib.hk_pages_free(ref, a, a, 3, None),
            lambda: lib.hk_pages_compact(ref, a, s, 1 << 40, None),
            lambda: lib.hk_pages_append(ref, 0, a, a, 128, a, a, 3, None),
            lambda: lib.hk_pages_attention(a, a, ref, 0, 8, 512, 512, a, a, 3, 100, s, 1 << 40, None)]


def refused(rc, text=b""):
    pk = package()
    assert rc == pk.hip_engine.HE_E_ARG
    message = pk.library().he_last_error()
    assert message.startswith(b"hk_") and text in message, message


@pytest.mark.parametrize("change, text", [
    (dict(head_size=80), b"head_size"), (dict(page_size=16), b"page_size"), (dict(page_size=48), b"page_size"),
    (dict(page_size=512), b"page_size"), (dict(n_layers=0), b"n_layers"), (dict(n_layers=1025), b"n_layers"),
    (dict(n_kv_heads=0), b"n_kv_heads"), (dict(n_kv_heads=1025), b"n_kv_heads"), (dict(n_pages=0), b"n_pages"),
    (dict(n_pages=(1 << 24) + 1), b"n_pages"), (dict(n_seqs=0), b"n_seqs"), (dict(n_seqs=8193), b"n_seqs"),
    (dict(table_size=0), b"table_size"), (dict(table_size=(1 << 24) + 1), b"table_size"),
    (dict(table_size=2147483647), b"table_size"), (dict(n_seqs=8192, page_size=32, table_size=131073), b"table_size")])
def test_caches_that_are_refused(change, text):
    lib, c = package().library(), made(**change)
    for call in calls(c):
        refused(call(), text)
    refused(lib.hk_pages_workspace(ctypes.byref(c)), text)
    refused(lib.hk_pages_attention_workspace(ctypes.byref(c), 8, 1, 1), text)


@pytest.mark.parametrize("name", ["keys", "values", "tables", "refs"])
def test_buffers_that_are_refused(name):
    for where in (None, (1 << 20) + 8):
        for call in calls(made(**{name: where})):
            refused(call(), b"buffer")
    for call in calls(None):
        refused(call(), b"null")


def test_lists_and_workspaces_that_are_refused():
    lib, c = package().library(), made()
    ref, a, s, need = ctypes.byref(c), 1 << 21, 1 << 24, lib.hk_pages_workspace(ctypes.byref(made()))
    assert need > 0
    for n in (0, -1, 8193):
        refused(lib.hk_pages_fork(ref, a, a, a, n, a, None), b"n is in")
        refused(lib.hk_pages_reserve(ref, a, a, a, n, a, s, need, None), b"n is in")
        refused(lib.hk_pages_free(ref, a, a, n, None), b"n is in")
    for bad in (None, a + 2):
        for i in range(3):
            lists = [a, a, a]
            lists[i] = bad
            refused(lib.hk_pages_fork(ref, *lists, 3, a, None), b"list")
            refused(lib.hk_pages_reserve(ref, *lists, 3, a, s, need, None), b"list")
        refused(lib.hk_pages_free(ref, bad, a, 3, None), b"list")
    refused(lib.hk_pages_fork(ref, a, a, a, 3, a + 2, None), b"status")
    refused(lib.hk_pages_reserve(ref, a, a, a, 3, a + 2, s, need, None), b"status")
    refused(lib.hk_pages_free(ref, a, a + 1, 3, None), b"4-byte")
    refused(lib.hk_pages_compact(ref, a + 2, s, need, None), b"used")
    for where, size in ((None, need), (s + 8, need), (s, need - 1)):
        refused(lib.hk_pages_reserve(ref, a, a, a, 3, a, where, size, None), b"workspace")
        refused(lib.hk_pages_compact(ref, a, where, size, None), b"workspace")


@pytest.mark.parametrize("change, text", [
    (dict(layer=-1), b"layer"), (dict(layer=2), b"layer"), (dict(k=None), b"k or v"), (dict(v=(1 << 21) + 4), b"16-byte"),
    (dict(stride=124), b"kv_stride"), (dict(stride=130), b"kv_stride"), (dict(positions=None), b"list"), (dict(seqs=(1 << 21) + 2), b"list"),
    (dict(n=0), b"n is in"), (dict(n=(1 << 20) + 1), b"n is in")])
def test_rows_that_are_refused(change, text):
    args = dict(layer=0, k=1 << 21, v=1 << 21, stride=128, seqs=1 << 21, positions=1 << 21, n=3)
    args.update(change)
    refused(package().library().hk_pages_append(ctypes.byref(made()), *args.values(), None), text)


@pytest.mark.parametrize("change, text", [
    (dict(out=None), b"out or q"), (dict(q=(1 << 21) + 4), b"16-byte"), (dict(layer=2), b"layer"), (dict(layer=-1), b"layer"),
    (dict(heads=7), b"n_heads"), (dict(heads=0), b"n_heads"), (dict(heads=66), b"n_heads"), (dict(q_stride=508), b"q_stride"),
    (dict(out_stride=514), b"out_stride"), (dict(lengths=None), b"list"), (dict(seqs=(1 << 21) + 2), b"list"), (dict(n=0), b"n is in"),
    (dict(n=65536), b"n is in"), (dict(longest=-1), b"longest"), (dict(longest=1281), b"longest")])
def test_attention_calls_that_are_refused(change, text):
    args = dict(layer=0, heads=8, q_stride=512, out_stride=512, seqs=1 << 21, lengths=1 << 21, n=3, longest=100)
    out, q = change.get("out", 1 << 21), change.get("q", 1 << 21)
    args.update({name: x for name, x in change.items() if name in args})
    refused(package().library().hk_pages_attention(out, q, ctypes.byref(made()), *args.values(), 1 << 24, 1 << 40, None), text)


def test_attention_workspaces_that_are_refused():
    lib, c = package().library(), made(table_size=100000, n_pages=100000)
    ref, a = ctypes.byref(c), 1 << 21
    need = lib.hk_pages_attention_workspace(ref, 8, 2, 200000)
    assert need > 0 and lib.hk_pages_attention_workspace(ref, 8, 2, 0) == 0
    for where, size in ((None, need), ((1 << 24) + 8, need), (1 << 24, need - 1)):
        refused(lib.hk_pages_attention(a, a, ref, 0, 8, 512, 512, a, a, 2, 200000, where, size, None), b"workspace")
    refused(lib.hk_pages_attention_workspace(ref, 7, 2, 100), b"n_heads")
    refused(lib.hk_pages_attention_workspace(ref, 8, 0, 100), b"n is in")
    refused(lib.hk_pages_attention_workspace(ref, 8, 65536, 100), b"n is in")
    refused(lib.hk_pages_attention_workspace(ref, 8, 2, -1), b"longest")
    refused(lib.hk_pages_attention_workspace(ref, 8, 2, 6400001), b"longest")


@pytest.mark.parametrize("half, heads, kv_heads, head_size", [(1, 8, 2, 64), (0, 32, 8, 128), (1, 1024, 1024, 16), (1, 32, 1, 256)])
def test_a_workspace_serves_every_smaller_call(half, heads, kv_heads, head_size):
    lib = package().library()
    ref = ctypes.byref(made(half=half, n_kv_heads=kv_heads, head_size=head_size, page_size=32, table_size=100000, n_pages=100000))
    rows, lengths = [1, 2, 31, 64, 255, 256, 257, 300, 5000, 65535], [0, 1, 640, 641, 1024, 1025, 2048, 2049, 50000, 3200000]
    need = [[lib.hk_pages_attention_workspace(ref, heads, n, longest) for longest in lengths] for n in rows]
    for i in range(len(rows)):
        for j in range(len(lengths)):
            assert need[i][j] >= (need[i - 1][j] if i else 0) and need[i][j] >= (need[i][j - 1] if j else 0)
            assert need[i][j] <= 1 << 33


@pytest.mark.parametrize("change, text", [
    (dict(m=0), b"m is in"), (dict(m=65536), b"m is in"), (dict(rows=0), b"rows"), (dict(rows=(1 << 26) + 1), b"rows"),
    (dict(k=0), b"k a multiple"), (dict(k=48), b"k a multiple"), (dict(k=(1 << 24) + 32), b"k a multiple"), (dict(bias=1), b"bias"),
    (dict(group=16), b"group"), (dict(group=256), b"group"), (dict(group=0), b"group"), (dict(y=None), b"pointer"),
    (dict(xq=None), b"pointer"), (dict(xs=None), b"pointer"), (dict(w=None), b"pointer"), (dict(ws=None), b"pointer"),
    (dict(w=(1 << 20) + 8), b"16-byte"), (dict(ws=(1 << 20) + 8), b"16-byte"), (dict(xq=(1 << 20) + 8), b"16-byte"),
    (dict(y=(1 << 20) + 2), b"4-byte"), (dict(xs=(1 << 20) + 1), b"4-byte")])
def test_products_that_are_refused(change, text):
    args = dict(y=1 << 20, xq=1 << 20, xs=1 << 20, w=1 << 20, ws=1 << 20, m=2, rows=10, k=64, bias=64, group=32, half=0)
    args.update(change)
    refused(package().library().hk_matmul_four(*args.values(), None), text)


def values(w, k):
    c = np.arange(k)
    byte, high = 64 * (c // 128) + 16 * (c // 4 % 4) + 4 * (c // 32 % 4) + c % 4, c // 16 % 2
    four = w[:, byte].astype(int) >> 4 * high & 15
    return np.where(four > 7, four - 16, four)


@pytest.mark.parametrize("group, half", [(32, False), (64, True), (128, False)])
@pytest.mark.parametrize("rows, k", [(1, 32), (5, 160), (3, 256)])
def test_quantized_rows(rows, k, group, half):
    x = np.random.default_rng(k).standard_normal((rows, k)).astype(np.float32)
    w, ws = package().quantize_four(x, group, half)
    wide = -(-k // 128) * 128
    assert w.shape == (rows, wide // 2) and w.dtype == np.uint8
    assert ws.shape == (rows, wide // group) and ws.dtype == (np.float16 if half else np.float32)
    q = values(w, wide)
    assert (q[:, k:] == 0).all()
    for r in range(rows):
        for g in range(-(-k // group)):
            part = x[r, g * group:(g + 1) * group]
            s = (np.abs(part).max() / np.float32(7)).astype(ws.dtype)
            assert s == ws[r, g]
            np.testing.assert_array_equal(q[r, g * group:g * group + len(part)],
                                          np.clip(np.rint(part.astype(np.float64) / np.float64(s)), -8, 7))


def test_rows_without_a_scale_are_zeros():
    x = np.zeros((4, 128), dtype=np.float32)
    x[1, 3], x[2, 40], x[3, 70] = np.inf, np.nan, 1e30
    w, ws = package().quantize_four(x, 32, True)
    assert (values(w, 128) == 0).all() and np.isfinite(ws).all()
    for bad in (np.zeros((2, 40)), np.zeros(32), np.zeros((0, 32))):
        with pytest.raises(ValueError):
            package().quantize_four(bad)
    with pytest.raises(ValueError):
        package().quantize_four(np.zeros((2, 64)), 48)
