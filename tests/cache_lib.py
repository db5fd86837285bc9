"""The cache held in 8 bits in NumPy (the oracle of hk_cache_*): its layout, its quantization in exact arithmetic, the
attention over it in float64, and the derived error of the kernels' float32 results."""
import ctypes

import numpy as np

from gpu_lib import Dev, check, hip, hip_check, upload
from paths import package

BLOCK, RECENT = 32, 128


def value_byte(t):
    return 16 * (t // 4 % 2) + 8 * (t // 16) + 4 * (t // 8 % 2) + t % 4


def quantize(x):
    """(int values, float32 scale) of a block's values of one head"""
    with np.errstate(invalid="ignore", divide="ignore"):
        s = np.float32(np.max(np.abs(x))) * np.float32(1 / 127)
        if not np.isfinite(s) or s == 0:
            return np.zeros(x.shape, dtype=np.int64), s
    return np.rint(x.astype(np.float64) / np.float64(s)).astype(np.int64), s


class Model:
    """what the cache holds after calls: float32 rows of every position, and the complete blocks in 8 bits"""

    def __init__(self, nkv, hs, seq_len):
        self.nkv, self.hs, self.seq_len = nkv, hs, seq_len
        self.rows = np.zeros((2, seq_len + BLOCK, nkv, hs), dtype=np.float32)
        self.q = np.zeros((2, -(-seq_len // BLOCK), nkv, BLOCK, hs), dtype=np.int64)
        self.s = np.zeros((2, -(-seq_len // BLOCK), nkv), dtype=np.float32)

    def append(self, k, v, pos):
        end = pos + len(k)
        for w, x in enumerate((k, v)):
            self.rows[w, pos:end] = x.reshape(len(k), self.nkv, self.hs)
            for b in range(pos // BLOCK, end // BLOCK):
                for h in range(self.nkv):
                    self.q[w, b, h], self.s[w, b, h] = quantize(self.rows[w, b * BLOCK:(b + 1) * BLOCK, h])

    def rewind(self, pos):
        first = pos // BLOCK * BLOCK
        self.rows[:, first:pos] = self.read(first, pos - first, 1 << 40).astype(np.float32)

    def eight(self, w, b):
        """block b's values as they stand, [32][nkv][hs]"""
        with np.errstate(invalid="ignore"):
            return (self.q[w, b] * self.s[w, b].astype(np.float64)[:, None, None]).transpose(1, 0, 2)

    def read(self, start, count, end):
        """positions start.. as a token at position end reads them, float64 [2][count][nkv][hs]"""
        out = np.zeros((2, count, self.nkv, self.hs))
        for w in range(2):
            for i in range(count):
                p = start + i
                out[w, i] = self.rows[w, p] if p // BLOCK == end // BLOCK else self.eight(w, p // BLOCK)[p % BLOCK]
        return out

    def attention(self, q, pos, nh):
        """(out, bound) [count][nh][hs]: the attention in float64, and how far a float32 result may lie from it.

        The bound, of a row with scores s and probabilities p: a query's digits are off by 0.5 / 4160000 of its largest
        value (rounded once), float32 products and sums by 2^-23 each, so a score by
        ds <= 2^-22 max|q| max_j sum|k_j| / sqrt(hs) + 2^-21 max|s| (nats: combined, scaled, the maximum taken off); a
        probability by 2 ds + 2^-21 (the exponential, two halves of 11 bits); and the float32 sums of n terms, 16 a
        product, by (n / 16 + 32) 2^-24: all of it at most that part of max|v|, three times over for the division by
        the sum and its own error."""
        count, hs, group = len(q), self.hs, nh // self.nkv
        out, off = np.zeros((count, nh, hs)), np.zeros((count, nh, hs))
        whole = (pos + count) // BLOCK + 1
        blocks = [[self.eight(w, b) if b < self.q.shape[1] else None for b in range(whole)] for w in range(2)]
        q = q.astype(np.float64).reshape(count, nh, hs)
        for i in range(count):
            p = pos + i
            first = p // BLOCK
            k, v = (np.concatenate(blocks[w][:first] + [self.rows[w, first * BLOCK:p + 1].astype(np.float64)])
                    for w in range(2))
            for h in range(nh):
                g = h // group
                s = k[:, g] @ q[i, h] / np.sqrt(hs)
                e = np.exp(s - s.max())
                out[i, h] = e @ v[:, g] / e.sum()
                ds = (2.0 ** -22 * np.abs(q[i, h]).max() * np.abs(k[:, g]).sum(-1).max() / np.sqrt(hs)
                      + 2.0 ** -21 * np.abs(s).max())
                n = len(s)
                off[i, h] = 3 * np.abs(v[:, g]).max() * (2 * ds + 2.0 ** -21 + (n / 16 + 32) * 2.0 ** -24)
        return out, off


class Cache:
    """a cache on the device (its buffers may start from a pattern, to see what calls leave alone)"""

    def __init__(self, nkv, hs, seq_len, fill=None):
        pk = package()
        self.nkv, self.hs, self.seq_len = nkv, hs, seq_len
        self.dev = {}
        for name, (shape, dtype) in pk.cache_shapes(nkv, hs, seq_len).items():
            init = None if fill is None else np.full(shape, fill if dtype != "float32" else fill / 7, dtype=dtype)
            self.dev[name] = Dev(shape, dtype, init)
        self.c = pk.HkCache(n_kv_heads=nkv, head_size=hs, seq_len=seq_len,
                            **{name: d.ptr.value for name, d in self.dev.items()})
        self.ref = ctypes.byref(self.c)

    def append(self, k, v, pos, stream=None):
        kd, vd = upload(k.astype(np.float32)), upload(v.astype(np.float32))
        check(package().library().hk_cache_append(self.ref, kd.ptr, vd.ptr, k.shape[1], len(k), pos, stream))
        hip_check(hip().hipDeviceSynchronize())

    def attention(self, q, k, v, pos, nh, pad=0):
        """the tokens' attention, with rows `pad` floats longer than they need to be on both sides"""
        lib, count, width = package().library(), len(q), nh * self.hs
        wide = np.full((count, width + pad), 5.0, dtype=np.float32)
        wide[:, :width] = q.reshape(count, width)
        rows = []
        for x in (k, v):
            r = np.full((count, self.nkv * self.hs + pad), 6.0, dtype=np.float32)
            r[:, :self.nkv * self.hs] = x.reshape(count, -1)
            rows.append(upload(r))
        qd, out = upload(wide), Dev((count, width + pad), np.float32, np.full((count, width + pad), 7.0))
        need = lib.hk_cache_workspace(self.ref, nh, count)
        assert need >= 0
        space = Dev(max(1, need), np.uint8, np.full(max(1, need), 0xFF))
        check(lib.hk_cache_attention(out.ptr, qd.ptr, rows[0].ptr, rows[1].ptr, self.ref, nh, width + pad,
                                     self.nkv * self.hs + pad, width + pad, count, pos, space.ptr, need, None))
        got = out.numpy()
        assert (got[:, width:] == 7.0).all()
        return got[:, :width].reshape(count, nh, self.hs)

    def rewind(self, pos):
        check(package().library().hk_cache_rewind(self.ref, pos, None))

    def read(self, start, count, end):
        out = [Dev((count, self.nkv, self.hs), np.float32) for _ in range(2)]
        check(package().library().hk_cache_read(out[0].ptr, out[1].ptr, self.ref, start, count, end, None))
        return np.stack([d.numpy() for d in out])

    def blocks(self):
        """the 8-bit values [2][blocks][nkv][32][hs] and scales [2][blocks][nkv] the buffers hold"""
        k = self.dev["keys"].numpy().transpose(1, 0, 3, 2, 4).reshape(-1, self.nkv, BLOCK, self.hs).astype(np.int64)
        v = self.dev["values"].numpy()[..., [value_byte(t) for t in range(BLOCK)]].astype(np.int64) - 128
        s = self.dev["scales"].numpy()
        return np.stack([k, v.transpose(1, 0, 3, 2)]), s.transpose(2, 1, 0)


def rows(rng, count, nkv, hs, wide=0.5):
    """keys and values as projections give them: channels of different size"""
    k = rng.standard_normal((count, nkv * hs)) * np.exp(wide * np.random.default_rng(1).standard_normal(nkv * hs))
    return k.astype(np.float32), rng.standard_normal((count, nkv * hs)).astype(np.float32)
