"""The 4-bit ICL cache in NumPy, float64, from its definition: what it holds,
its bytes, its bounds, the choice of blocks and the attention."""

import numpy as np

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def unit(largest, most, low, high):
    """The smallest 2^e, low <= e <= high, with largest <= most * 2^e (2^high when none)."""
    e = np.full(largest.shape, low)
    for power in range(low, high):
        e = np.where(largest > most * 2.0 ** power, power + 1, e)
    return e


def inside(shape, lengths):
    """[E, N]: the rows inside each estimator's length."""
    e, _, n = shape
    return np.arange(n) < (np.full(e, n) if lengths is None else np.minimum(lengths, n))[:, None]


def codes(x, axis):
    """Codes and exponents of x [..., N, 64] (N a multiple of 64), groups of 32 along axis."""
    groups = np.moveaxis(x, axis, -1)
    groups = groups.reshape(groups.shape[:-1] + (-1, 32))
    e = unit(np.abs(groups).max(-1), 6.0, -13, 13)
    m = np.minimum(np.abs(groups) / 2.0 ** e[..., None], 6.0)  # saturated
    distance = np.abs(m[..., None] - LEVELS)
    near = distance.argmin(-1)  # the lower of two
    tie = np.take_along_axis(distance, np.minimum(near + 1, 7)[..., None], -1)[..., 0] == distance.min(-1)
    c = np.where(tie & (near % 2 == 1) & (near < 7), near + 1, near) + 8 * (groups < 0)
    c = c.reshape(c.shape[:-2] + (-1,))
    return np.moveaxis(c, -1, axis), np.moveaxis(e, -1, axis)


def values(c, e, axis):
    table = np.concatenate((LEVELS, -LEVELS))
    return table[c] * 2.0 ** np.repeat(e, 32, axis=axis)


class Cache:
    """Held keys k and values v [E, H, T * 64, 64], bounds [E, H, T, 2, 64]
    (whole numbers) and their units [E, H, 64]."""

    def __init__(self, k, v, lengths=None):
        e, h, n, _ = k.shape
        self.shape, tiles = (e, h, n), -(-n // 64)
        self.lengths = lengths
        self.nonfinite = 0
        padded = []
        for x in (k, v):
            x = np.where(inside(self.shape, lengths)[:, None, :, None], x.astype(np.float64), 0.0)
            self.nonfinite += int((~np.isfinite(x)).sum())
            x = np.where(np.isfinite(x), x, 0.0)
            padded.append(np.concatenate((x, np.zeros((e, h, tiles * 64 - n, 64))), axis=2))
        self.kc, self.ke = codes(padded[0], 3)
        self.vc, self.ve = codes(padded[1], 2)
        self.k, self.v = values(self.kc, self.ke, 3), values(self.vc, self.ve, 2)
        x = unit(np.abs(self.k).max(2), 127.0, -20, 20)
        self.units = 2.0 ** x
        self.bounds = np.zeros((e, h, tiles, 2, 64))
        for i in range(e):
            rows = int(inside(self.shape, lengths)[i].sum())
            for t in range(-(-rows // 64)):
                block = self.k[i, :, 64 * t:min(rows, 64 * t + 64)] / self.units[i, :, None]
                self.bounds[i, :, t, 0], self.bounds[i, :, t, 1] = np.floor(block.min(1)), np.ceil(block.max(1))

    def bytes(self):
        """The cache's bytes, element by element from the stated positions."""
        e, h, n = self.shape
        pairs, tiles = e * h, -(-n // 64)
        out = np.zeros((pairs, tiles, 4352), np.uint8)
        r, d = np.meshgrid(np.arange(64), np.arange(64), indexing="ij")
        s = r // 32
        a, b, i = r // 16 % 2, r // 8 % 2, r % 8
        key_at = s * 1024 + ((d // 16 * 2 + a) * 8 + i) * 16 + b * 8 + d % 16 // 2
        t, b2, hh, j = r // 16 % 2, r // 8 % 2, r // 4 % 2, r % 4
        value_at = 2048 + s * 1024 + ((t * 2 + hh) * 16 + d % 16) * 16 + d // 16 * 4 + b2 * 2 + j // 2
        kc, vc = (c.reshape(pairs, tiles, 64, 64).astype(np.uint8) for c in (self.kc, self.vc))
        for p in range(pairs):
            for tile in range(tiles):
                np.bitwise_or.at(out[p, tile], key_at, kc[p, tile] << (4 * (d % 2)).astype(np.uint8))
                np.bitwise_or.at(out[p, tile], value_at, vc[p, tile] << (4 * (j % 2)).astype(np.uint8))
        r, u = np.meshgrid(np.arange(64), np.arange(2), indexing="ij")
        out[:, :, 4096 + ((u * 2 + r // 16 % 2) * 8 + r % 8) * 4 + r // 32 * 2 + r // 8 % 2] = \
            (self.ke + 127).reshape(pairs, tiles, 64, 2)
        s, d = np.meshgrid(np.arange(2), np.arange(64), indexing="ij")
        out[:, :, 4224 + d % 16 * 8 + s * 4 + d // 16] = (self.ve + 127).reshape(pairs, tiles, 2, 64)
        return np.concatenate((out.ravel(), self.bounds.astype(np.int8).view(np.uint8).ravel(),
                               self.units.astype(np.float32).view(np.uint8).ravel()))

    def attended(self, keep=None):
        """[E, T * 64]: the rows that queries attend to."""
        rows = inside(self.shape, self.lengths)
        rows = rows if keep is None else rows & keep
        return np.concatenate((rows, np.zeros((rows.shape[0], self.k.shape[2] - rows.shape[1]), bool)), axis=1)

    def scores(self, q):
        """[E, H, Q, T] whole numbers."""
        x = q.astype(np.float64) * self.units[:, :, None]
        c = np.rint(x / 2.0 ** unit(np.abs(x).max(-1), 127.0, -100, 200)[..., None])
        # The sum over dims of max(c low, c high), one dim at a time.
        total = np.zeros(q.shape[:3] + (self.bounds.shape[2],))
        for d in range(64):
            low, high = self.bounds[:, :, None, :, 0, d], self.bounds[:, :, None, :, 1, d]
            total += np.maximum(c[..., d, None] * low, c[..., d, None] * high)
        return total

    def select(self, q, n, keep=None):
        some = self.attended(keep).reshape(self.shape[0], -1, 64).any(-1)
        scores = np.where(some[:, None, None], self.scores(q), -np.inf)
        order = np.argsort(-scores, axis=-1, kind="stable")[..., :n]
        tiles = scores.shape[-1]
        order = np.where(np.take_along_axis(scores, order, -1) == -np.inf, tiles, order)
        order = np.sort(order, axis=-1)
        out = np.full(q.shape[:3] + (n,), -1, np.int32)
        out[..., : order.shape[-1]] = np.where(order == tiles, -1, order)
        return out

    def attend(self, q, scale=0.125, keep=None, blocks=None):
        """Output, log-sum-exp, and the largest sum over dims of |scale q k| (for tolerances)."""
        q = q.astype(np.float64)
        weight = np.broadcast_to(self.attended(keep)[:, None, None], q.shape[:3] + (self.k.shape[2],)).astype(float)
        if blocks is not None:
            tiles = self.k.shape[2] // 64
            times = np.zeros(q.shape[:3] + (tiles,))
            for e, h, r, i in np.ndindex(*blocks.shape):
                if 0 <= blocks[e, h, r, i] < tiles:
                    times[e, h, r, blocks[e, h, r, i]] += 1
            weight = weight * np.repeat(times, 64, axis=-1)
        scores = np.matmul(q, self.k.swapaxes(2, 3)) * scale
        with np.errstate(divide="ignore"):
            scores = scores + np.log(weight)
        largest = scores.max(-1, keepdims=True)
        largest = np.where(np.isfinite(largest), largest, 0.0)
        p = np.exp(scores - largest)
        total = p.sum(-1, keepdims=True)
        out = np.matmul(p, self.v) / np.where(total == 0, 1.0, total)
        with np.errstate(divide="ignore"):
            lse = (largest + np.log(total))[..., 0]
        return out, lse, (np.matmul(np.abs(q), np.abs(self.k).swapaxes(2, 3)) * scale).max()


def bits(keep):
    """[E, N] truth values as the words that `keep` takes."""
    e, n = keep.shape
    padded = np.zeros((e, -(-n // 64) * 64), np.uint8)
    padded[:, :n] = keep
    return np.packbits(padded, axis=1, bitorder="little").view(np.uint64)
