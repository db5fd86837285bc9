"""Oracles of hk_pages_attention over long rows that see a single position: queries of zero, under which the result is the mean of
the values to the bit; and for any queries a bound that goes by the outputs' own size."""
import numpy as np

from pages_lib import filled

U = 2.0 ** -24  # of a value, a float32 rounding


def whole(rng, layers, nkv, page, hs, half, lengths):
    """pages_lib.filled with values that are whole numbers in 0..15"""
    model = filled(rng, layers, nkv, page, hs, half, lengths)
    model.values[:] = rng.integers(0, 16, model.values.shape)
    return model


def means(model, layer, seqs, lengths, nh):
    """the attention of queries of zero [rows][nh][hs]: all scores 0, all probabilities 1, their sum the length, the weighted sums
    whole numbers below 2^24 (and their multiples by 64 of as many bits), which float32 holds whatever the order of the additions.
    So the one rounding is the division's"""
    sums, out = {}, np.zeros((len(lengths), nh, model.hs), dtype=np.float32)
    for i, n in enumerate(lengths):
        s = i if seqs is None else seqs[i]
        if n <= 0 or s < 0:
            continue
        if s not in sums:
            most = max(m for j, m in enumerate(lengths) if (j if seqs is None else seqs[j]) == s)
            _, v = model.rows(layer, s, most)
            sums[s] = np.cumsum(v, axis=0)
            assert sums[s].max() < 1 << 24
        out[i] = np.repeat(sums[s][n - 1].astype(np.float32) / np.float32(n), nh // model.nkv, axis=0)
    return out


def close(model, layer, q, seqs, lengths, nh, adds):
    """(out, bound) [rows][nh][hs] in float64, for rows of at least one position.

    A score j is off by d_j = (hs + 8) u sum|q k_j| / sqrt(hs) + 4 u |s_j| (as in Model.attention), its probability by that and
    2^-21 of itself (the exponential, halves of 2^-23). That moves the result by sum p_j (d_j + 2^-21) |v_j - out| / sum p.
    `adds` is how many additions an accumulator takes on the way: each a rounding of at most u sum p |v| / sum p, above the
    division and below it. A hundredth more for products of such errors."""
    out, off = np.zeros((len(q), nh, model.hs)), np.zeros((len(q), nh, model.hs))
    q = q.astype(np.float64).reshape(len(q), nh, model.hs)
    for i, n in enumerate(lengths):
        k, v = model.rows(layer, i if seqs is None else seqs[i], n)
        for h in range(nh):
            g = h // (nh // model.nkv)
            x = k[:, g] @ q[i, h] / np.sqrt(model.hs)
            p = np.exp(x - x.max())
            p /= p.sum()
            out[i, h] = p @ v[:, g]
            d = (model.hs + 8) * U * (np.abs(k[:, g]) @ np.abs(q[i, h])) / np.sqrt(model.hs) + 4 * U * np.abs(x) + 2.0 ** -21
            off[i, h] = 1.01 * ((p * d) @ np.abs(v[:, g] - out[i, h]) + 2 * adds * U * (p @ np.abs(v[:, g])))
    return out, off
