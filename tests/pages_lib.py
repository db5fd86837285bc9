"""The cache in pages in NumPy (the oracle of hk_pages_*): its tables, counts and pools after calls, the attention over it in
float64 with the derived error of the kernels' float32 results; and the device's side of the same calls."""
import ctypes

import numpy as np

from gpu_lib import Dev, check, hip, hip_check, upload
from paths import package


class Model:
    def __init__(self, layers, pages, nkv, page, hs, half, seqs, slots, rng=None):
        self.layers, self.pages, self.nkv, self.page, self.hs, self.half, self.seqs, self.slots = (layers, pages, nkv, page, hs,
                                                                                                   half, seqs, slots)
        shapes = package().pages_shapes(layers, pages, nkv, page, hs, half, seqs, slots)
        made = {name: np.full(shape, start, dtype=dtype) for name, (shape, dtype, start) in shapes.items()}
        self.keys, self.values, self.tables, self.refs = made["keys"], made["values"], made["tables"], made["refs"]
        if rng is not None:  # rows that nothing has written: anything
            for pool in (self.keys, self.values):
                pool[:] = rng.standard_normal(pool.shape, dtype=np.float32)

    def lists_hold(self, seqs, *numbers):
        most = self.slots * self.page
        listed = [i for i, s in enumerate(seqs) if s >= 0]
        if len({seqs[i] for i in listed}) < len(listed):
            return False
        return all(seqs[i] < self.seqs and all(0 <= x[i] <= most for x in numbers) for i in listed)

    def fork(self, to, source, lengths):
        if not self.lists_hold(to, lengths) or any(not 0 <= f < self.seqs for t, f in zip(to, source) if t >= 0):
            return -1
        before = self.tables.copy()
        for t, f, n in zip(to, source, lengths):
            if t >= 0:
                held = -(-n // self.page)
                self.tables[t, :held] = before[f, :held]
                self.tables[t, held:] = -1
        self.refs[:] = np.bincount(self.tables[self.tables >= 0], minlength=self.pages)
        return 0

    def reserve(self, seqs, starts, ends):
        if not self.lists_hold(seqs, starts, ends):
            return -1
        asked = []
        for s, a, b in zip(seqs, starts, ends):
            if s >= 0 and b > a:
                for slot in range(a // self.page, (b - 1) // self.page + 1):
                    old = self.tables[s, slot]
                    if old < 0 or self.refs[old] > 1:
                        asked.append((s, slot, old, a - slot * self.page))
        free = np.flatnonzero(self.refs == 0)
        if len(free) < len(asked):
            return len(asked) - len(free)
        for (s, slot, old, kept), new in zip(asked, free):
            self.tables[s, slot] = new
            if old >= 0 and kept > 0:
                for pool in (self.keys, self.values):
                    pool[:, new, :, :kept] = pool[:, old, :, :kept]
        self.refs[:] = np.bincount(self.tables[self.tables >= 0], minlength=self.pages)
        return 0

    def free(self, seqs, kept=None):
        for i, s in enumerate(seqs):
            if 0 <= s < self.seqs:
                self.tables[s, max(0, -(-(kept[i] if kept is not None else 0) // self.page)):] = -1
        self.refs[:] = np.bincount(self.tables[self.tables >= 0], minlength=self.pages)

    def compact(self):
        used = int((self.refs > 0).sum())
        holes = np.flatnonzero(self.refs[:used] == 0)
        moved = used + np.flatnonzero(self.refs[used:] > 0)
        place = np.arange(self.pages, dtype=np.int32)
        place[moved] = holes
        for pool in (self.keys, self.values):
            pool[:, holes] = pool[:, moved]
        self.tables[:] = np.where(self.tables >= 0, place[self.tables], -1)
        self.refs[:] = np.bincount(self.tables[self.tables >= 0], minlength=self.pages)
        return used

    def append(self, layer, k, v, seqs, positions):
        for i, (s, p) in enumerate(zip(seqs, positions)):
            if 0 <= s < self.seqs and 0 <= p < self.slots * self.page and self.tables[s, p // self.page] >= 0:
                with np.errstate(over="ignore"):
                    for pool, x in ((self.keys, k), (self.values, v)):
                        pool[layer, self.tables[s, p // self.page], :, p % self.page] = x[i].reshape(self.nkv, self.hs)

    def rows(self, layer, seq, n):
        """keys and values of the first n positions, float64 [n][nkv][hs]"""
        held = self.tables[seq, :-(-n // self.page)]
        return (pool[layer, held].transpose(0, 2, 1, 3).reshape(-1, self.nkv, self.hs)[:n].astype(np.float64)
                for pool in (self.keys, self.values))

    def attention(self, layer, q, seqs, lengths, nh):
        """(out, bound) [rows][nh][hs]: the attention in float64, and how far a float32 result may lie from it.

        The bound, with u = 2^-24 of a value a float32 operation's rounding: a score is at most hs + 8 of them off its sum of
        magnitudes (products in float32 order, the queries' halves 1, scaled, the reference taken off: 2 of the scores
        themselves), ds = (hs + 8) u max_j sum|q k_j| / sqrt(hs) + 4 u max|s|; a probability is off by its score's error
        (nats) and 2^-21 (the exponential, its halves); a sum over n positions by as many roundings as one accumulator takes,
        n / 2 + 64 at most. All of it of max|v|, twice: above and below the division."""
        out, off, u = np.zeros((len(q), nh, self.hs)), np.zeros((len(q), nh, self.hs)), 2.0 ** -24
        q = q.astype(np.float64).reshape(len(q), nh, self.hs)
        for i, n in enumerate(lengths):
            s = i if seqs is None else seqs[i]
            if n <= 0 or s < 0:
                continue
            k, v = self.rows(layer, s, n)
            for h in range(nh):
                g = h // (nh // self.nkv)
                x = k[:, g] @ q[i, h] / np.sqrt(self.hs)
                e = np.exp(x - x.max())
                out[i, h] = e @ v[:, g] / e.sum()
                ds = (self.hs + 8) * u * (np.abs(k[:, g]) @ np.abs(q[i, h])).max() / np.sqrt(self.hs) + 4 * u * np.abs(x).max()
                off[i, h] = 2 * np.abs(v[:, g]).max() * (ds + 2.0 ** -21 + (n / 2 + 64) * u)
        return out, off


def ints(values):
    return upload(np.asarray(values, dtype=np.int32)) if values is not None else None


def at(dev):
    return dev.ptr if dev is not None else None


class Pages:
    """the same cache on the device, from a model's present state"""

    def __init__(self, model):
        self.m = model
        self.dev = {name: upload(getattr(model, name)) for name in ("keys", "values", "tables", "refs")}
        self.c = package().HkPages(n_layers=model.layers, n_pages=model.pages, n_kv_heads=model.nkv, page_size=model.page,
                                   head_size=model.hs, half=int(model.half), n_seqs=model.seqs, table_size=model.slots,
                                   **{name: d.ptr.value for name, d in self.dev.items()})
        self.ref, self.lib = ctypes.byref(self.c), package().library()
        need = self.lib.hk_pages_workspace(self.ref)
        self.space, self.need = upload(np.full(need, 0xA5, dtype=np.uint8)), need

    def same(self):
        for name in ("tables", "refs"):
            np.testing.assert_array_equal(self.dev[name].numpy(), getattr(self.m, name), err_msg=name)
        bits = np.uint16 if self.m.half else np.uint32
        for name in ("keys", "values"):
            got, want = self.dev[name].numpy().view(bits), getattr(self.m, name).view(bits)
            assert (got == want).all(), (name, np.argwhere(got != want)[:4])

    def status(self, call, lists, *more):
        devs, out = [ints(x) for x in lists], ints([77])
        check(call(self.ref, *(at(d) for d in devs), len(lists[0]), out.ptr, *more, None))
        return int(out.numpy()[0])

    def fork(self, to, source, lengths):
        return self.status(self.lib.hk_pages_fork, (to, source, lengths))

    def reserve(self, seqs, starts, ends):
        return self.status(self.lib.hk_pages_reserve, (seqs, starts, ends), self.space.ptr, self.need)

    def free(self, seqs, kept=None):
        s, k = ints(seqs), ints(kept)
        check(self.lib.hk_pages_free(self.ref, s.ptr, at(k), len(seqs), None))
        hip_check(hip().hipDeviceSynchronize())

    def compact(self):
        used = ints([77])
        check(self.lib.hk_pages_compact(self.ref, used.ptr, self.space.ptr, self.need, None))
        return int(used.numpy()[0])

    def append(self, layer, k, v, seqs, positions, pad=0):
        width = self.m.nkv * self.m.hs
        devs = []
        for x in (k, v):
            wide = np.full((len(x), width + pad), 9.0, dtype=np.float32)
            wide[:, :width] = x.reshape(len(x), width)
            devs.append(upload(wide))
        s, p = ints(seqs), ints(positions)
        check(self.lib.hk_pages_append(self.ref, layer, devs[0].ptr, devs[1].ptr, width + pad, at(s), p.ptr, len(positions), None))
        hip_check(hip().hipDeviceSynchronize())

    def attention(self, layer, q, seqs, lengths, nh, longest=None, pad=0):
        n, width = len(q), nh * self.m.hs
        longest = max(0, max(lengths)) if longest is None else longest
        wide = np.full((n, width + pad), 5.0, dtype=np.float32)
        wide[:, :width] = q.reshape(n, width)
        qd, out = upload(wide), upload(np.full((n, width + pad), 7.0, dtype=np.float32))
        need = self.lib.hk_pages_attention_workspace(self.ref, nh, n, longest)
        assert need >= 0
        space = upload(np.full(max(1, need), 0xFF, dtype=np.uint8))  # (NaN, should any of it be read unwritten)
        s, lens = ints(seqs), ints(lengths)
        check(self.lib.hk_pages_attention(out.ptr, qd.ptr, self.ref, layer, nh, width + pad, width + pad, at(s), lens.ptr, n,
                                          longest, space.ptr, need, None))
        got = out.numpy()
        assert (got[:, width:] == 7.0).all()
        return got[:, :width].reshape(n, nh, self.m.hs)


def filled(rng, layers, nkv, page, hs, half, lengths, spare=3, slots=None):
    """a model whose sequences hold `lengths` positions, in pages of no order, and every row drawn"""
    held = [-(-n // page) for n in lengths]
    model = Model(layers, sum(held) + spare, nkv, page, hs, half, len(lengths), slots or max(max(held), 1) + 1, rng)
    order = rng.permutation(model.pages)
    first = 0
    for s, n in enumerate(held):
        model.tables[s, :n] = order[first:first + n]
        first += n
    model.refs[:] = np.bincount(model.tables[model.tables >= 0], minlength=model.pages)
    return model


def within(got, model, layer, q, seqs, lengths, nh):
    want, off = model.attention(layer, q, seqs, lengths, nh)
    assert np.isfinite(got).all()
    bad = np.abs(got - want) > off
    assert not bad.any(), (np.argwhere(bad)[:4], np.abs(got - want).max(), off.min())
