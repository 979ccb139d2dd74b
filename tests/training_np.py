"""Attention for training, its backward pass and dropout in float64 NumPy, from their definitions."""

import numpy as np

M0, M1, W0, W1 = 0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85  # Salmon, Moraes, Dror and Shaw, SC 2011
LOW = np.uint64(0xFFFFFFFF)


def philox(counter, key, rounds=7):
    """Four uint64 arrays of words below 2^32."""
    c = [np.asarray(x, np.uint64) for x in counter]
    k = [int(x) for x in key]
    for _ in range(rounds):
        a, b = c[0] * np.uint64(M0), c[2] * np.uint64(M1)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & LOW, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & LOW]
        k = [(k[0] + W0) & 0xFFFFFFFF, (k[1] + W1) & 0xFFFFFFFF]
    return c


def values(counter, seed, index):
    """The 16-bit value `index` (0 to 7) of each counter's call."""
    words = np.stack(np.broadcast_arrays(*philox(np.broadcast_arrays(*counter), (seed & 0xFFFFFFFF, seed >> 32))))
    word = np.take_along_axis(words, np.broadcast_to(index // 2, words.shape[1:])[None], axis=0)[0]
    return (word >> np.uint64(16) * (index % 2).astype(np.uint64)) & np.uint64(0xFFFF)


def kept_weights(seed, site, dropped, pair, q_rows, rows):
    """[q_rows, rows] truth values: the weights of (estimator, head) `pair` that stay."""
    if not dropped:
        return np.ones((q_rows, rows), bool)
    j, i = np.arange(rows)[None, :], np.arange(q_rows)[:, None]
    cell = 2 * (j // 16) + j // 4 % 2
    index = np.broadcast_to(4 * (j // 8 % 2) + j % 4, (q_rows, rows))
    return values((cell, i, np.full_like(j, pair), np.full_like(j, site)), seed, index) >= np.uint64(dropped)


def kept_numbers(seed, site, dropped, rows, width):
    """[rows, width] truth values of dropout."""
    if not dropped:
        return np.ones((rows, width), bool)
    j, i = np.arange(width)[None, :], np.arange(rows)[:, None]
    index = np.broadcast_to(j % 8, (rows, width))
    return values((j // 8, i, np.full_like(j, 0xFFFFFFFF), np.full_like(j, site)), seed, index) >= np.uint64(dropped)


def bits(keep):
    """[E, N] truth values as 64-bit words, row r at bit r % 64 of word r / 64."""
    e, n = keep.shape
    padded = np.zeros((e, -(-n // 64), 64), np.uint8)
    padded.reshape(e, -1)[:, :n] = keep
    return np.packbits(padded, axis=-1, bitorder="little").view(np.uint64)[..., 0]


def terms(factor, rows):
    """[2, results, 1] of factors [results, terms] and rows [terms, 64]."""
    largest = np.abs(rows).max(-1)
    return np.stack(((factor * largest).max(-1), factor.max(-1) * largest.max()))[..., None]


class Attention:
    """float64 results and, for error bounds, sums of magnitudes of every output. Inputs [E, H, Q, 64] and [E, G, N, 64]."""

    def __init__(self, q, k, v, scale=0.125, q_lengths=None, lengths=None, keep=None, seed=0, site=0, dropped=0, dout=None):
        q, k, v = (x.astype(np.float64) for x in (q, k, v))
        e, h, m, _ = q.shape
        g, n = k.shape[1:3]
        w = 65536.0 / (65536 - dropped)
        self.out, self.lse = np.zeros(q.shape), np.full((e, h, m), -np.inf)
        self.r, self.s = np.zeros((e, h, m)), np.zeros((e, h, m))
        self.magnitude, self.out_abs = np.zeros((e, h, m)), np.zeros(q.shape)
        self.dq, self.dq_abs = np.zeros(q.shape), np.zeros(q.shape)
        self.dk, self.dv, self.dk_abs, self.dv_abs = (np.zeros(k.shape) for _ in range(4))
        # The largest |factor| times its row's largest number among a result's terms, and the largest factor times the largest
        # number of all rows.
        self.out_term, self.dq_term = np.zeros((2, e, h, m, 1)), np.zeros((2, e, h, m, 1))
        self.dk_term, self.dv_term = np.zeros((2, e, g, n, 1)), np.zeros((2, e, g, n, 1))
        self.inside = np.arange(m) < (np.full(e, m) if q_lengths is None else np.minimum(q_lengths, m))[:, None]
        self.held = np.arange(n) < (np.full(e, n) if lengths is None else np.minimum(lengths, n))[:, None]
        self.attended = self.held if keep is None else self.held & keep
        for i in range(e):
            rows, queries = np.flatnonzero(self.attended[i]), np.flatnonzero(self.inside[i])
            if not len(rows) or not len(queries):
                continue
            for j in range(h):
                kk, vv, qq = k[i, j // (h // g), rows], v[i, j // (h // g), rows], q[i, j, queries]
                x = qq @ kk.T * scale
                top = x.max(-1, keepdims=True)
                p = np.exp(x - top)
                total = p.sum(-1, keepdims=True)
                self.lse[i, j, queries] = (top + np.log(total))[:, 0]
                r = np.ceil(top * np.log2(np.e))
                self.r[i, j, queries] = r[:, 0]
                self.s[i, j, queries] = (total * np.exp2(top * np.log2(np.e) - r))[:, 0]
                p = p / total
                z = kept_weights(seed, site, dropped, i * h + j, m, n)[np.ix_(queries, rows)] * w
                size = np.abs(qq) @ np.abs(kk).T * scale
                self.magnitude[i, j, queries] = size.max(-1)
                self.out[i, j, queries] = (p * z) @ vv
                self.out_abs[i, j, queries] = (p * z) @ np.abs(vv)
                self.out_term[:, i, j, queries] = terms(p * w, vv)
                if dout is None:
                    continue
                d = dout[i, j, queries].astype(np.float64)
                o = self.out[i, j, queries]
                dp, dp_abs = d @ vv.T * z, np.abs(d) @ np.abs(vv).T * z
                delta, delta_abs = (d * o).sum(-1, keepdims=True), (np.abs(d) * self.out_abs[i, j, queries]).sum(-1, keepdims=True)
                ds, ds_abs = p * (dp - delta), p * (dp_abs + delta_abs)
                self.dq[i, j, queries] = ds @ kk * scale
                self.dq_abs[i, j, queries] = ds_abs @ np.abs(kk) * scale
                self.dk[i, j // (h // g), rows] += ds.T @ qq * scale
                self.dq_term[:, i, j, queries] = terms(ds_abs, kk) * scale
                for into, factor, of in ((self.dk_term, ds_abs * scale, qq), (self.dv_term, p * w, d)):
                    into[:, i, j // (h // g), rows] = np.maximum(into[:, i, j // (h // g), rows], terms(factor.T, of))
                self.dk_abs[i, j // (h // g), rows] += ds_abs.T @ np.abs(qq) * scale
                self.dv[i, j // (h // g), rows] += (p * z).T @ d
                self.dv_abs[i, j // (h // g), rows] += (p * z).T @ np.abs(d)
