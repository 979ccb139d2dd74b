"""The 4-bit ICL cache on the GPU against its definition in float64
(icl4_np.py): what it holds bit for bit, the choice of blocks exactly, the
attention within bounds worked out beforehand.

Bounds. A score is a sum of 64 products: FP32 queries as pairs of FP16 values
are off by at most 2^-22 relative each, a 64-term FP32 sum by 2^-18 of the sum
of magnitudes A, and FP32's scaling by less: |ds| <= 2^-17 A. (One or two queries'
31-bit integers are off by 2^-31 of its largest number, those of more than 16
by 2^-24 of it, or for FP16 by 2^-19 where they are below 2^-9 of it. The
largest of 64 normal numbers is at most 6 times the mean of their sizes, and
some one in a hundred is that small: 2^-21 and 2^-22 of A, inside the half of
the bound that the sum leaves.) A weight exp(s) is
then off by 2 ds relative, and so is a weighted mean of values up to V by at
most 4 ds V (numerator and denominator). FP32 weights are pairs (2^-22); FP16
ones are off by half a step, 2^-11, and below FP16's smallest step (half of it
2^-25, where the largest weight is at least 2^5) by at most 2^-30 of the
largest, N of them. FP32 sums of N / 8 addends (two keys' worth of
products in one) add N 2^-27 V at most. FP16 outputs round by 2^-11 of
themselves. The log-sum-exp is off by 2 ds, N 2^-27 and 2^-22 of itself.

FP16 numbers of more than 16 queries a call are rounded from 2^-8 of the largest down, not from 2^-9: two in a hundred
normal ones, 2^-21 of A, inside the same half. A query that this, or FP32's 2^-24, could cost 2^-14 of a score and 2^-20
of the sum of the sizes of |scale q| times the largest |k| is rounded more finely."""

import ctypes

import numpy as np
import pytest

import icl4_np
from ironicl_amd import hip, hipmem, icl4

pytestmark = pytest.mark.gpu
DTYPES = {"f32": np.float32, "f16": np.float16}


@pytest.fixture(scope="module")
def device():
    return hip.Device(0)


def put(a):
    return None if a is None else hipmem.DeviceArray.from_host(np.ascontiguousarray(a))


class Tensor:
    """[E, H, N, 64] on the device, head-major or as token rows [E, N, H * 64 + gap]."""

    def __init__(self, shape, element, layout="heads", host=None):
        e, h, n, _ = shape
        self.shape, self.layout, self.element = shape, layout, element
        self.width = h * 64 + 16  # token rows with a gap
        if layout == "heads":
            self.strides, full = (h * n * 64, n * 64, 64), (e, h, n, 64)
        else:
            self.strides, full = (n * self.width, 64, self.width), (e, n, self.width)
        self.host = np.full(full, 77, DTYPES[element])
        if host is not None:
            self.view(self.host)[:] = host
        self.array = put(self.host)

    def view(self, a):
        if self.layout == "heads":
            return a
        e, h, n, _ = self.shape
        return a[:, :, : h * 64].reshape(e, n, h, 64).transpose(0, 2, 1, 3) if a is not self.host else \
            np.lib.stride_tricks.as_strided(a, self.shape, [s * a.itemsize for s in self.strides] + [a.itemsize])

    def get(self):
        a = self.array.to_host()
        if self.layout != "heads":
            assert np.all(a[:, :, self.shape[1] * 64:] == 77), "written past the heads"
        return np.ascontiguousarray(self.view(a))


def draw(shape, element, seed, scale=1.0):
    return (np.random.default_rng(seed).standard_normal(shape) * scale).astype(DTYPES[element])


def make(device, e, h, n, element="f32", layout="heads", lengths=None, seed=0, k=None, v=None):
    """A cache on the device and its definition, from random (or the given) keys and values."""
    k = draw((e, h, n, 64), element, seed, 1.3) if k is None else k
    v = draw((e, h, n, 64), element, seed + 1) if v is None else v
    want = icl4_np.Cache(k, v, lengths)
    dk, dv = (Tensor(x.shape, element, layout, x) for x in (k, v))
    cache = hipmem.DeviceArray((icl4.cache_bytes((e, h, n)),), np.uint8)
    bad = put(np.array([5], np.uint32))
    icl4.encode(device, (e, h, n), dk.array, dv.array, cache, element=element, k_strides=dk.strides,
                v_strides=dv.strides, lengths=put_lengths(lengths), nonfinite=bad)
    hipmem.synchronize()
    assert int(bad.to_host()[0]) == 5 + want.nonfinite
    return cache, want


KEPT = []  # small device arrays of calls whose work may still run


def put_lengths(lengths):
    if lengths is None:
        return None
    KEPT.append(put(np.asarray(lengths, np.uint32)))
    return KEPT[-1]


def workspace(device, shape, q_rows, n_blocks=0):
    size = icl4.workspace_bytes(device, shape, q_rows, n_blocks)
    # Full of NaN: nothing may hang on what it held.
    return {"workspace": put(np.full(max(size, 16), 255, np.uint8)), "workspace_bytes": size}


def attend(device, cache, shape, q, element="f32", layout="heads", keep=None, lengths=None, blocks=None, scale=0.125):
    rows = q.shape[2]
    dq, out = Tensor(q.shape, element, layout, q), Tensor(q.shape, element, layout)
    lse = put(np.full(q.shape[:3], 77, np.float32))
    n = 0 if blocks is None else blocks.shape[-1]
    words = None if keep is None else put(icl4_np.bits(keep))
    space, listed, rows_of = workspace(device, shape, rows, n), put(blocks), put_lengths(lengths)
    icl4.attention(device, shape, cache, dq.array, rows, out.array, element=element, scale=scale, q_strides=dq.strides,
                   out_strides=out.strides, lengths=rows_of, keep=words, blocks=listed, n_blocks=n, lse=lse, **space)
    hipmem.synchronize()
    return out.get(), lse.to_host()


def select(device, cache, shape, q, n, element="f32", layout="heads", keep=None, lengths=None):
    dq = Tensor(q.shape, element, layout, q)
    out = put(np.full(q.shape[:3] + (n,), 77, np.int32))
    words, rows_of = None if keep is None else put(icl4_np.bits(keep)), put_lengths(lengths)
    space = workspace(device, shape, q.shape[2], n)
    icl4.select(device, shape, cache, dq.array, q.shape[2], n, out, element=element, q_strides=dq.strides,
                lengths=rows_of, keep=words, **space)
    hipmem.synchronize()
    return out.to_host()


def check(got, want, element, cache):
    (out, lse), (out64, lse64, magnitude) = got, want
    ds = 2.0 ** -17 * magnitude
    n, v = cache.k.shape[2], np.abs(cache.v).max()
    weight = 2.0 ** -21 if element == "f32" else 2.0 ** -10
    bound = v * (4 * ds + weight + n * 2.0 ** -27 + n * 2.0 ** -30)
    if element == "f16":
        bound = bound + np.abs(out64) * 2.0 ** -11 + 2.0 ** -25
    assert np.isfinite(out).all()
    off = np.abs(out.astype(np.float64) - out64) - bound
    assert off.max() <= 0, f"{off.max():.3e} past the bound"
    empty = np.isneginf(lse64)
    assert np.array_equal(np.isneginf(lse), empty)
    assert np.all(out[empty] == 0)
    off = np.abs(lse[~empty] - lse64[~empty]) - (2 * ds + n * 2.0 ** -26 + 2.0 ** -21 * np.abs(lse64[~empty]) + 1e-6)
    assert empty.all() or off.max() <= 0, f"lse {off.max():.3e} past the bound"


# ---- what the cache holds ----

@pytest.mark.parametrize("e,h,n,element,layout,lengths", [
    (1, 1, 1, "f32", "heads", None),
    (1, 8, 63, "f32", "heads", None),
    (1, 8, 64, "f16", "tokens", None),
    (2, 3, 65, "f32", "tokens", (65, 2)),
    (3, 8, 200, "f16", "heads", (0, 200, 129)),
    (2, 5, 130, "f32", "heads", (1000, 64)),
    (2, 2, 2047, "f32", "heads", (2047, 700)),
    (2, 2, 2049, "f16", "tokens", (2049, 700)),
    (1, 1, 70001, "f32", "heads", None),
])
def test_cache_holds_what_it_says(device, e, h, n, element, layout, lengths):
    print(f"encode {e} x {h} x {n} {element} {layout} {lengths}", flush=True)
    cache, want = make(device, e, h, n, element, layout, lengths)
    np.testing.assert_array_equal(cache.to_host(), want.bytes())
    outs = [Tensor((e, h, n, 64), element, layout) for _ in range(2)]
    bounds = put(np.full((e * h, -(-n // 64), 2, 64), 77, np.float32))
    icl4.decode(device, (e, h, n), cache, outs[0].array, outs[1].array, element=element, k_strides=outs[0].strides,
                v_strides=outs[1].strides, lengths=put_lengths(lengths), bounds=bounds)
    hipmem.synchronize()
    rows = icl4_np.inside((e, h, n), lengths)[:, None, :, None]
    for out, held in zip(outs, (want.k, want.v)):
        np.testing.assert_array_equal(out.get(), np.where(rows, held[:, :, :n], 77))  # rows past the length stay
    np.testing.assert_array_equal(bounds.to_host(),
                                  (want.bounds * want.units[:, :, None, None]).reshape(e * h, -1, 2, 64))


@pytest.mark.parametrize("element", ["f32", "f16"])
def test_cache_of_odd_numbers(device, element):
    """Ties, both zeros, subnormals, the largest numbers, infinities and NaN, and rows of zeros."""
    levels = np.array([0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, -0.25, -0.75, -5.0, -0.0, 0.2501, 4.999, 5.001])
    rng = np.random.default_rng(3)
    k, v = (levels[rng.integers(0, 16, (1, 2, 150, 64))] * 2.0 ** rng.integers(-18, 13, (1, 2, 150, 1))
            for _ in range(2))
    k[0, 0, 3] = 0.0
    k[0, 0, 4, :5] = (np.inf, -np.inf, np.nan, 3.0, 65504.0)
    k[0, 1, 7, 40] = 1e-7
    v[0, 0, 64:96, 7] = 0.0
    v[0, 1, 100, :4] = (np.nan, np.inf, -65504.0, 65504.0)
    k, v = k.astype(DTYPES[element]), v.astype(DTYPES[element])
    if element == "f32":
        k[0, 1, 9, :3] = (3e38, -1e30, 1e-40)
        v[0, 0, 20, 9] = -3.4e38
    cache, want = make(device, 1, 2, 150, element, k=k, v=v)
    assert want.nonfinite == 5
    got = cache.to_host()
    # A negative number that rounds to zero may be held as either zero: compared by value below.
    outs = [Tensor((1, 2, 150, 64), "f32") for _ in range(2)]
    icl4.decode(device, (1, 2, 150), cache, outs[0].array, outs[1].array)
    hipmem.synchronize()
    for out, held in zip(outs, (want.k, want.v)):
        np.testing.assert_array_equal(out.get(), held[:, :, :150])
    np.testing.assert_array_equal(got[2 * 3 * 4352:], want.bytes()[2 * 3 * 4352:])


def test_one_side_is_read_alone(device):
    cache, want = make(device, 1, 2, 70)
    out = Tensor((1, 2, 70, 64), "f16", "tokens")
    icl4.decode(device, (1, 2, 70), cache, v=out.array, element="f16", v_strides=out.strides)
    hipmem.synchronize()
    np.testing.assert_array_equal(out.get(), want.v[:, :, :70])


# ---- attention ----

@pytest.mark.parametrize("element,layout", [("f32", "heads"), ("f16", "tokens"), ("f32", "tokens"), ("f16", "heads")])
@pytest.mark.parametrize("e,h,n,rows", [(1, 8, 1, 1), (1, 8, 63, 3), (2, 4, 64, 16), (1, 8, 65, 17), (1, 3, 1000, 1),
                                        (2, 8, 777, 33), (1, 8, 2049, 65), (1, 2, 640, 130), (1, 1, 5000, 300),
                                        (1, 2, 20011, 5), (1, 8, 1025, 2), (1, 3, 20011, 1)])
def test_attention(device, e, h, n, rows, element, layout):
    print(f"attention {e} x {h} x {n}, {rows} queries, {element} {layout}", flush=True)
    cache, want = make(device, e, h, n, element, layout, seed=n)
    q = draw((e, h, rows, 64), element, n + 7, 1.5)
    check(attend(device, cache, (e, h, n), q, element, layout), want.attend(q), element, want)


@pytest.mark.parametrize("element", ["f32", "f16"])
@pytest.mark.parametrize("rows", [1, 20, 150, 600])
def test_attention_of_ragged_and_masked_estimators(device, element, rows):
    """Lengths 0, 1, odd, past the rows; masks that leave blocks, single rows and nothing."""
    e, h, n = 6, 2, 700
    lengths = (0, 1, 333, 9999, 700, 700)
    keep = np.random.default_rng(rows).random((e, n)) < 0.5
    keep[3, 128:512] = False
    keep[4] = False
    keep[5] = False
    keep[5, 130] = True
    cache, want = make(device, e, h, n, element, lengths=lengths, seed=5)
    q = draw((e, h, rows, 64), element, 11, 1.5)
    got = attend(device, cache, (e, h, n), q, element, keep=keep, lengths=lengths)
    check(got, want.attend(q, keep=keep), element, want)
    assert np.all(got[0][0] == 0) and np.all(got[0][4] == 0)
    # One attended row: its held value, whatever its score.
    bound = np.abs(want.v[5, :, None, 130]) * (2.0 ** -20 if element == "f32" else 2.0 ** -11)
    assert np.all(np.abs(got[0][5] - want.v[5, :, None, 130]) <= bound)


@pytest.mark.parametrize("element", ["f32", "f16"])
@pytest.mark.parametrize("rows", [1, 2, 3, 16])
def test_few_queries_of_ragged_and_masked_estimators(device, element, rows):
    """Splits of long contexts, some of them past an estimator's length or masked whole."""
    e, h, n = 4, 2, 9001
    lengths = (9001, 0, 1500, 9000)
    keep = np.random.default_rng(rows).random((e, n)) < 0.5
    keep[0, 640:5000] = False
    keep[3, :8990] = False
    cache, want = make(device, e, h, n, element, lengths=lengths, seed=6)
    q = draw((e, h, rows, 64), element, 12, 1.5)
    check(attend(device, cache, (e, h, n), q, element, keep=keep, lengths=lengths), want.attend(q, keep=keep), element, want)


def test_keep_bits_past_the_rows_are_not_read_as_rows(device):
    cache, want = make(device, 1, 2, 70)
    q = draw((1, 2, 4, 64), "f32", 1)
    words = put(np.full((1, 2), 2 ** 64 - 1, np.uint64))
    out = Tensor(q.shape, "f32")
    dq, space = put(q), workspace(device, (1, 2, 70), 4)
    icl4.attention(device, (1, 2, 70), cache, dq, 4, out.array, keep=words, **space)
    hipmem.synchronize()
    np.testing.assert_allclose(out.get(), want.attend(q)[0], atol=1e-4)


@pytest.mark.parametrize("rows", [2, 70])
@pytest.mark.parametrize("element", ["f32", "f16"])
def test_attention_of_peaked_and_extreme_scores(device, element, rows):
    """A later key far above the first ones, keys and values of the largest and smallest held sizes, large and zero
    queries, and a scale that is not 1 / 8."""
    n = 900
    k, v = draw((1, 2, n, 64), element, 1), draw((1, 2, n, 64), element, 2)
    k[0, 0, 500:] *= 8
    k[0, 1, 700] *= 40
    v[0, :, 100:140] *= 2.0 ** 14
    v[0, :, 140:180] *= 2.0 ** -12
    cache, want = make(device, 1, 2, n, element, k=k, v=v)
    q = draw((1, 2, rows, 64), element, 3)
    q[0, 0, 0] = 0.0
    q[0, 1, 1] *= 30
    if element == "f32":
        q[0, 0, 1] *= 1e-30
    check(attend(device, cache, (1, 2, n), q, element, scale=0.3), want.attend(q, scale=0.3), element, want)


@pytest.mark.parametrize("element", ["f32", "f16"])
@pytest.mark.parametrize("rows,listed", [(1, False), (2, False), (5, False), (70, False), (2100, False), (5, True)])
def test_scores_past_what_fp32_tells_apart(device, element, rows, listed):
    """Scores of 2^18 to 2^40, where FP32's step is 2^-5 to 2^17. Two equal keys lie far above the others (8 times their
    scores and more), so each query gets the mean of their values, with two equal weights w. As pairs they and their
    products are off by 2^-20 of the values. Rounded to FP16 both are off by the same 2^-11 at most, and the sum of
    weights that divides them is not rounded: 2^-11 of the mean, and the output's rounding as much again. The
    log-sum-exp is the score and log 2, off by 2^-19 of it."""
    e, h, n = 2, 8, 900
    rng = np.random.default_rng(rows)
    k = rng.choice([-0.5, 0.5, 1.0], (e, h, n, 64)).astype(DTYPES[element])
    k[:, :, 333] = k[:, :, 800] = 8.0
    v = draw((e, h, n, 64), element, 3)
    cache, want = make(device, e, h, n, element, k=k, v=v)
    expected = (want.v[:, :, None, 333] + want.v[:, :, None, 800]) / 2
    bound = np.abs(expected) * 2.0 ** -19 + np.abs(want.v).max() * 2.0 ** -20
    if element == "f16":
        bound = bound + np.abs(expected) * 2.0 ** -10 + 2.0 ** -25
    size = 2.0 ** rng.uniform(0, 8, (e, h, rows, 1))
    q = np.broadcast_to(size, (e, h, rows, 64)).astype(DTYPES[element])
    tiles = -(-n // 64)
    blocks = np.broadcast_to(np.arange(tiles, dtype=np.int32), (e, h, rows, tiles)) if listed else None
    for power in (9, 16, 23, 31):
        scale = 2.0 ** power
        out, lse = attend(device, cache, (e, h, n), q, element, blocks=blocks, scale=scale)
        assert np.all(np.abs(out - expected) <= bound), power
        total = q[..., 0].astype(np.float64) * 512 * scale + np.log(2.0)
        assert np.all(np.abs(lse - total) <= total * 2.0 ** -19), power


@pytest.mark.parametrize("element", ["f32", "f16"])
@pytest.mark.parametrize("e,h,n,rows,listed", [(1, 2, 20011, 1, 0), (1, 2, 20011, 2, 0), (1, 2, 20011, 5, 0),
                                               (2, 1, 20011, 16, 0), (1, 2, 20011, 70, 0), (2, 8, 9001, 2100, 0),
                                               (1, 2, 70000, 3, 1000)])
def test_large_equal_scores_in_different_splits(device, e, h, n, rows, listed, element):
    """Seven equal keys in the first block and one in the last, which another split takes, at scores of 2^16 to 2^31:
    eight equal weights, whatever plan the sizes get. Bounds as for two of them: pairs and eight FP32 sums of products
    are off by 2^-20 of the values, FP16 weights all by the same 2^-11, and the output's rounding by as much again."""
    assert icl4.workspace_bytes(device, (e, h, n), rows, listed) > 0
    rng = np.random.default_rng(rows)
    k = rng.choice([-0.5, 0.5, 1.0], (e, h, n, 64)).astype(DTYPES[element])
    tied = np.r_[2:63:10, n - 3]
    k[:, :, tied] = 8.0
    v = draw((e, h, n, 64), element, 3)
    cache, want = make(device, e, h, n, element, k=k, v=v)
    expected = want.v[:, :, None, tied].mean(3)
    bound = np.abs(expected) * 2.0 ** -19 + np.abs(want.v).max() * 2.0 ** -20
    if element == "f16":
        bound = bound + np.abs(expected) * 2.0 ** -10 + 2.0 ** -25
    q = np.broadcast_to(rng.uniform(1, 2, (e, h, rows, 1)), (e, h, rows, 64)).astype(DTYPES[element])
    blocks = None
    if listed:
        tiles = -(-n // 64)
        blocks = np.broadcast_to(np.r_[0:listed - 1, tiles - 1].astype(np.int32), (e, h, rows, listed))
    for power in (7, 12, 17, 21):
        scale = 2.0 ** power
        out, lse = attend(device, cache, (e, h, n), q, element, blocks=blocks, scale=scale)
        assert np.all(np.abs(out - expected) <= bound), power
        total = q[..., 0].astype(np.float64) * 512 * scale + np.log(8.0)
        assert np.all(np.abs(lse - total) <= total * 2.0 ** -19), power


@pytest.mark.parametrize("element", ["f32", "f16"])
@pytest.mark.parametrize("n,rows,listed", [(20011, 1, 0), (20011, 5, 0), (20011, 70, 0), (70000, 3, 1000)])
def test_a_query_that_is_not_a_number_stays_alone_in_splits(device, n, rows, listed, element):
    assert icl4.workspace_bytes(device, (1, 2, n), rows, listed) > 0
    cache, _ = make(device, 1, 2, n, element)
    q = draw((1, 2, rows, 64), element, 4)
    blocks = np.broadcast_to(np.arange(listed, dtype=np.int32), (1, 2, rows, listed)) if listed else None
    whole, whole_lse = attend(device, cache, (1, 2, n), q, element, blocks=blocks)
    for bad in (np.nan, np.inf):
        q[0, 1, rows - 1, 9] = bad
        got, lse = attend(device, cache, (1, 2, n), q, element, blocks=blocks)
        others = np.ones((1, 2, rows), bool)
        others[0, 1, rows - 1] = False
        np.testing.assert_array_equal(got[others], whole[others])
        np.testing.assert_array_equal(lse[others], whole_lse[others])
        assert np.isnan(got[0, 1, rows - 1]).all() and np.isnan(lse[0, 1, rows - 1])


@pytest.mark.parametrize("element", ["f32", "f16"])
@pytest.mark.parametrize("e,rows,listed", [(2, 1, False), (2, 16, False), (2, 20, False), (2, 70, False),
                                           (16, 2100, False), (2, 5, True)])
def test_zero_queries_at_the_smallest_scales(device, e, rows, listed, element):
    """The mean of the attended values and the logarithm of their number, beside masked rows, rows past the last and a
    query that is not zero."""
    h, n = 1 if e == 16 else 2, 900
    keep = np.random.default_rng(1).random((e, n)) < 0.7
    keep[:, 640:768] = True
    cache, want = make(device, e, h, n, element)
    tiles = -(-n // 64)
    blocks = np.broadcast_to(np.arange(tiles, dtype=np.int32), (e, h, rows, tiles)) if listed else None
    q = np.zeros((e, h, rows, 64), DTYPES[element])
    q[:, :, 1::7] = 0.5
    for scale in (1e-13, 1e-16, 1e-30, 1e-38, 1e-45):
        got = attend(device, cache, (e, h, n), q, element, keep=keep, blocks=blocks, scale=scale)
        check(got, want.attend(q, scale=scale, keep=keep, blocks=blocks), element, want)


@pytest.mark.parametrize("rows,listed", [(1, 0), (3, 0), (16, 0), (40, 0), (600, 0), (5, 13), (9000, 3)])
@pytest.mark.parametrize("power", [90, 99, 105, 112, 120, 126])
def test_tiny_fp32_queries(device, rows, listed, power):
    """Queries near FP32's smallest numbers (their smaller ones below its smallest normal number), with a scale that
    brings their scores back: bit for bit what the same queries times 2^power give at a scale of 1/8."""
    cache, want = make(device, 1, 2, 900)
    q = np.ldexp(draw((1, 2, rows, 64), "f32", 4, 1.5).astype(np.float64), -power).astype(np.float32)
    blocks = np.random.default_rng(5).integers(0, 15, (1, 2, rows, listed)).astype(np.int32) if listed else None
    scale = 0.125 * 2.0 ** power
    got = attend(device, cache, (1, 2, 900), q, blocks=blocks, scale=scale)
    back = np.ldexp(q.astype(np.float64), power).astype(np.float32)
    whole = attend(device, cache, (1, 2, 900), back, blocks=blocks)
    np.testing.assert_array_equal(got[0], whole[0])
    np.testing.assert_array_equal(got[1], whole[1])
    some = np.r_[0:rows:37, rows - 1]
    check((got[0][:, :, some], got[1][:, :, some]),
          want.attend(q[:, :, some], scale=scale, blocks=None if blocks is None else blocks[:, :, some]), "f32", want)


@pytest.mark.parametrize("rows,listed", [(1, 0), (3, 0), (40, 0), (5, 13)])
def test_the_largest_fp32_queries_at_scales_below_the_smallest_normal_number(device, rows, listed):
    """A scale of two bits, whose product with log2 e has more."""
    cache, want = make(device, 1, 2, 900, k=draw((1, 2, 900, 64), "f32", 3, 4096.0))
    q = np.ldexp(draw((1, 2, rows, 64), "f32", 4, 1.5).astype(np.float64), 124).astype(np.float32)
    blocks = np.random.default_rng(5).integers(0, 15, (1, 2, rows, listed)).astype(np.int32) if listed else None
    scale = 3 * 2.0 ** -149
    got = attend(device, cache, (1, 2, 900), q, blocks=blocks, scale=scale)
    check(got, want.attend(q, scale=scale, blocks=blocks), "f32", want)


@pytest.mark.parametrize("element", ["f32", "f16"])
@pytest.mark.parametrize("rows,listed", [(1, 0), (3, 0), (40, 0), (5, 13)])
def test_zero_queries_at_the_largest_scale(device, rows, listed, element):
    cache, want = make(device, 1, 2, 900, element)
    q = np.zeros((1, 2, rows, 64), DTYPES[element])
    blocks = np.random.default_rng(5).integers(0, 15, (1, 2, rows, listed)).astype(np.int32) if listed else None
    got = attend(device, cache, (1, 2, 900), q, element, blocks=blocks, scale=2.0 ** 127)
    check(got, want.attend(q, blocks=blocks), element, want)


@pytest.mark.parametrize("element", ["f32", "f16"])
@pytest.mark.parametrize("e,h,n,rows,listed", [(1, 2, 900, 1, 0), (1, 2, 900, 16, 0), (1, 2, 900, 17, 0),
                                               (1, 3, 5000, 70, 0), (16, 1, 900, 2100, 0), (1, 2, 900, 20, 14)])
@pytest.mark.parametrize("outlier", [2000.0, 8000.0, 30000.0])
def test_queries_with_one_large_channel(device, e, h, n, rows, listed, element, outlier):
    """A number 1,000 to 20,000 times the others, whose keys are zero: scores are the others' sums, and neither they nor
    their bound may lose bits to it. Some queries have none, and one has a second number between."""
    k = draw((e, h, n, 64), element, 1, 1.3)
    k[..., 40] = 0.0
    cache, want = make(device, e, h, n, element, k=k)
    q = draw((e, h, rows, 64), element, 2, 1.5)
    q[:, :, ::3, 40] = outlier
    q[:, :, rows // 2, 40] = -outlier / 3
    q[:, :, rows // 2, 7] = 31.0
    blocks = np.broadcast_to(np.arange(listed, dtype=np.int32), (e, h, rows, listed)) if listed else None
    out, lse = attend(device, cache, (e, h, n), q, element, blocks=blocks)
    some = np.r_[0:rows:37, rows // 2, rows - 1]
    check((out[:, :, some], lse[:, :, some]),
          want.attend(q[:, :, some], blocks=None if blocks is None else blocks[:, :, some]), element, want)


@pytest.mark.parametrize("rows", [16, 17, 40])
def test_the_last_bit_of_a_small_fp16_number(device, rows):
    """2^-8 (1 + 2^-10) beside 2, on a key of 49,152: a score of 192.1875 against one of 192."""
    k, v = np.zeros((1, 1, 70, 64), np.float16), draw((1, 1, 70, 64), "f16", 3)
    k[0, 0, 0, 5], k[0, 0, 69, 40] = 49152, 192
    cache, want = make(device, 1, 1, 70, "f16", k=k, v=v)
    q = np.zeros((1, 1, rows, 64), np.float16)
    q[..., 1], q[..., 5], q[..., 40] = 2, 2.0 ** -8 + 2.0 ** -18, 1
    check(attend(device, cache, (1, 1, 70), q, "f16", scale=1.0), want.attend(q, scale=1.0), "f16", want)


@pytest.mark.parametrize("element,rows", [("f32", 70), ("f16", 70), ("f16", 2100)])
def test_a_query_with_one_large_channel_leaves_the_others(device, element, rows):
    """Bit for bit, whatever the form does for it."""
    cache, _ = make(device, 2, 8, 900, element)
    q = draw((2, 8, rows, 64), element, 2, 1.5)
    whole, whole_lse = attend(device, cache, (2, 8, 900), q, element)
    q[:, :, 5::32, 40] = 30000.0
    got, lse = attend(device, cache, (2, 8, 900), q, element)
    others = np.arange(rows) % 32 != 5
    np.testing.assert_array_equal(got[:, :, others], whole[:, :, others])
    np.testing.assert_array_equal(lse[:, :, others], whole_lse[:, :, others])


@pytest.mark.parametrize("e,rows,listed", [(2, 1, 0), (2, 16, 0), (2, 20, 0), (2, 70, 0), (16, 2100, 0), (2, 5, 13),
                                           (2, 6000, 3)])
@pytest.mark.parametrize("power", [12, 20])
def test_subnormal_fp16_queries(device, e, rows, listed, power):
    """Bit for bit what the same queries times 2^power give at a scale of 1/8."""
    h, n = 1 if e == 16 else 2, 900
    keep = np.random.default_rng(1).random((e, n)) < 0.8
    cache, want = make(device, e, h, n, "f16")
    q = np.ldexp(draw((e, h, rows, 64), "f32", 4, 1.5).astype(np.float64), -power).astype(np.float16)
    blocks = np.random.default_rng(5).integers(0, 15, (e, h, rows, listed)).astype(np.int32) if listed else None
    scale = 0.125 * 2.0 ** power
    got = attend(device, cache, (e, h, n), q, "f16", keep=keep, blocks=blocks, scale=scale)
    back = np.ldexp(q.astype(np.float64), power).astype(np.float16)
    whole = attend(device, cache, (e, h, n), back, "f16", keep=keep, blocks=blocks)
    np.testing.assert_array_equal(got[0], whole[0])
    np.testing.assert_array_equal(got[1], whole[1])
    some = np.r_[0:rows:37, rows - 1]
    check((got[0][:, :, some], got[1][:, :, some]),
          want.attend(q[:, :, some], scale=scale, keep=keep, blocks=None if blocks is None else blocks[:, :, some]),
          "f16", want)


@pytest.mark.parametrize("element", ["f32", "f16"])
@pytest.mark.parametrize("rows,blocks", [(1, 0), (16, 0), (70, 0), (3, 900)])
def test_splits_of_any_lengths(device, rows, blocks, element):
    """Lengths around the splits' ends, one at 1 and one at 0: splits that hold nothing, and those that hold one row."""
    n, e = 20011, 6
    lengths = (0, 1, 63, 64, 65, 19969)
    keep = np.ones((e, n), bool)
    keep[5, ::2] = False
    cache, want = make(device, e, 1, n, element, lengths=lengths, seed=3)
    assert icl4.workspace_bytes(device, (e, 1, n), rows, blocks) > 0
    q = draw((e, 1, rows, 64), element, 4, 1.5)
    listed = None
    if blocks:
        listed = np.random.default_rng(2).integers(-3, 330, (e, 1, rows, blocks)).astype(np.int32)
        listed[..., 0] = 0
    got = attend(device, cache, (e, 1, n), q, element, keep=keep, lengths=lengths, blocks=listed)
    check(got, want.attend(q, keep=keep, blocks=listed), element, want)
    assert np.all(got[0][0] == 0) and np.all(np.isneginf(got[1][0]))


@pytest.mark.parametrize("element", ["f32", "f16"])
@pytest.mark.parametrize("e,h,n,rows", [(1, 2, 900, 20), (1, 2, 20011, 70), (16, 1, 900, 2100)])
def test_large_scores_of_queries_with_one_large_channel(device, e, h, n, rows, element):
    """Scores of 2^16 to 2^31 by 63 channels, and a number of 30,000 on keys of zero in every other query. Bounds as for
    equal scores in different splits."""
    rng = np.random.default_rng(rows)
    k = rng.choice([-0.5, 0.5, 1.0], (e, h, n, 64)).astype(DTYPES[element])
    tied = np.r_[2:63:10, n - 3]
    k[:, :, tied] = 8.0
    k[..., 40] = 0.0
    v = draw((e, h, n, 64), element, 3)
    cache, want = make(device, e, h, n, element, k=k, v=v)
    expected = want.v[:, :, None, tied].mean(3)
    bound = np.abs(expected) * 2.0 ** -19 + np.abs(want.v).max() * 2.0 ** -20
    if element == "f16":
        bound = bound + np.abs(expected) * 2.0 ** -10 + 2.0 ** -25
    q = np.broadcast_to(rng.uniform(1, 2, (e, h, rows, 1)), (e, h, rows, 64)).astype(DTYPES[element])
    q[:, :, ::2, 40] = 30000.0
    for power in (7, 12, 17, 21):
        scale = 2.0 ** power
        out, lse = attend(device, cache, (e, h, n), q, element, scale=scale)
        assert np.all(np.abs(out - expected) <= bound), power
        total = q[..., 0].astype(np.float64) * 504 * scale + np.log(8.0)
        assert np.all(np.abs(lse - total) <= total * 2.0 ** -19), power


def test_large_fp32_queries(device):
    """Queries past FP16's range, with a scale that brings their scores back."""
    cache, want = make(device, 1, 8, 300)
    q = draw((1, 8, 40, 64), "f32", 4) * np.float32(1e6)
    for rows in (3, 40):
        got = attend(device, cache, (1, 8, 300), q[:, :, :rows], scale=1e-7)
        check(got, want.attend(q[:, :, :rows], scale=1e-7), "f32", want)


def test_a_query_that_is_not_finite_leaves_the_others(device):
    cache, _ = make(device, 1, 8, 300)
    q = draw((1, 8, 70, 64), "f32", 4)
    whole, _ = attend(device, cache, (1, 8, 300), q)
    q[0, 3, 5, 9] = np.nan
    got, _ = attend(device, cache, (1, 8, 300), q)
    others = np.ones((1, 8, 70), bool)
    others[0, 3, 5] = False
    np.testing.assert_array_equal(got[others], whole[others])
    assert np.isnan(got[0, 3, 5]).all()


@pytest.mark.parametrize("element", ["f32", "f16"])
@pytest.mark.parametrize("rows,listed", [(1, False), (5, False), (70, False), (5, True)])
def test_a_query_that_is_not_a_number_stays_alone(device, element, rows, listed):
    cache, _ = make(device, 2, 4, 700, element)
    q = draw((2, 4, rows, 64), element, 4)
    blocks = np.broadcast_to(np.arange(0, 10, 2, dtype=np.int32), (2, 4, rows, 5)) if listed else None
    whole, whole_lse = attend(device, cache, (2, 4, 700), q, element, blocks=blocks)
    q[1, 2, rows - 1, 9] = np.nan
    got, lse = attend(device, cache, (2, 4, 700), q, element, blocks=blocks)
    others = np.ones((2, 4, rows), bool)
    others[1, 2, rows - 1] = False
    np.testing.assert_array_equal(got[others], whole[others])
    np.testing.assert_array_equal(lse[others], whole_lse[others])
    assert np.isnan(got[1, 2, rows - 1]).all() and np.isnan(lse[1, 2, rows - 1])


@pytest.mark.parametrize("element,rows", [("f32", 1568), ("f16", 2109), ("f16", 1570)])
def test_attention_of_more_queries_than_the_gpu_takes_at_once(device, element, rows):
    """Units of work past a whole round of workgroups, of which the last ones are split; every 37th query is checked."""
    e, h, n = 2, 8, 2500
    lengths = (2500, 2203)
    keep = np.random.default_rng(rows).random((e, n)) < 0.9
    cache, want = make(device, e, h, n, element, lengths=lengths, seed=8)
    q = draw((e, h, rows, 64), element, 9, 1.5)
    out, lse = attend(device, cache, (e, h, n), q, element, keep=keep, lengths=lengths)
    some = np.r_[0:rows:37, rows - 2:rows]
    check((out[:, :, some], lse[:, :, some]), want.attend(q[:, :, some], keep=keep), element, want)
    assert np.isfinite(out).all() and np.isfinite(lse).all()


# ---- the choice of blocks, and attention over it ----

@pytest.mark.parametrize("element,layout", [("f32", "heads"), ("f16", "tokens")])
@pytest.mark.parametrize("e,h,n,rows,count", [(1, 8, 1, 1, 1), (1, 8, 640, 3, 4), (2, 3, 1000, 20, 16), (1, 2, 130, 5, 9),
                                              (1, 2, 20011, 3, 100), (1, 1, 70000, 2, 700), (2, 8, 777, 150, 1)])
def test_select(device, e, h, n, rows, count, element, layout):
    print(f"select {count} of {e} x {h} x {n}, {rows} queries, {element} {layout}", flush=True)
    cache, want = make(device, e, h, n, element, layout, seed=n)
    q = draw((e, h, rows, 64), element, n + 3, 1.5)
    np.testing.assert_array_equal(select(device, cache, (e, h, n), q, count, element, layout), want.select(q, count))


def test_select_of_equal_scores_takes_the_lower_blocks(device):
    """Every block the same rows, and queries of zeros."""
    k = np.tile(draw((1, 2, 64, 64), "f32", 1), (1, 1, 40, 1))
    cache, want = make(device, 1, 2, 2560, k=k, v=k)
    q = draw((1, 2, 6, 64), "f32", 2)
    q[0, :, 3:] = 0.0
    got = select(device, cache, (1, 2, 2560), q, 7)
    np.testing.assert_array_equal(got, want.select(q, 7))
    assert np.all(got == np.arange(7))


@pytest.mark.parametrize("times,rows", [(3, 70), (30, 2), (30, 40)])
def test_select_of_many_blocks(device, times, rows):
    """500 blocks over and over: 1,500 for many queries and 15,000, in the forms that keep scores in memory. Equal
    scores are many, and the lowest of them are taken."""
    k = draw((1, 2, 32000, 64), "f32", 5)
    want = icl4_np.Cache(k, k)
    whole, shape = np.tile(k, (1, 1, times, 1)), (1, 2, 32000 * times)
    cache = hipmem.DeviceArray((icl4.cache_bytes(shape),), np.uint8)
    dk = put(whole)
    icl4.encode(device, shape, dk, dk, cache)
    hipmem.synchronize()
    q = draw((1, 2, 300 if times == 3 else rows, 64), "f32", 6)
    keep = np.random.default_rng(7).random((1, shape[2] // 64)) < 0.8
    scores = np.where(keep[:, None, None], np.tile(want.scores(q), (1, 1, 1, times)), -np.inf)
    order = np.sort(np.argsort(-scores, axis=-1, kind="stable")[..., :rows], axis=-1)
    got = select(device, cache, shape, q, rows, keep=np.repeat(keep, 64, axis=1))
    np.testing.assert_array_equal(got, order)


def test_select_of_masked_and_empty_blocks(device):
    e, h, n = 4, 2, 900
    lengths = (0, 65, 900, 500)
    keep = np.random.default_rng(1).random((e, n)) < 0.3
    keep[2, 64:640] = False
    keep[3, 1:] = False
    cache, want = make(device, e, h, n, lengths=lengths)
    q = draw((e, h, 5, 64), "f32", 2)
    for count in (1, 6, 15, 40):
        got = select(device, cache, (e, h, n), q, count, keep=keep, lengths=lengths)
        np.testing.assert_array_equal(got, want.select(q, count, keep=keep))
    assert np.all(got[0] == -1) and np.all(got[3, :, :, 1:] == -1)


@pytest.mark.parametrize("e,h,tiles,rows,count", [(1, 2, 256, 40, 9), (2, 1, 257, 33, 17), (1, 1, 700, 17, 100),
                                                  (1, 1, 960, 16, 960), (1, 1, 961, 17, 100), (1, 1, 512, 16, 512),
                                                  (1, 1, 513, 17, 100), (1, 2, 600, 1024, 9), (1, 2, 960, 1009, 960),
                                                  (1, 2, 961, 1009, 100)])
def test_select_on_both_sides_of_its_forms(device, e, h, tiles, rows, count):
    n = 64 * tiles - 5
    lengths = (n, n - 1000)[:e]
    keep = np.random.default_rng(tiles).random((e, n)) < 0.02
    cache, want = make(device, e, h, n, "f16", lengths=lengths, seed=tiles)
    q = draw((e, h, rows, 64), "f16", 2)
    got = select(device, cache, (e, h, n), q, count, "f16", keep=keep, lengths=lengths)
    np.testing.assert_array_equal(got, want.select(q, count, keep=keep))


def test_select_of_queries_of_any_size(device):
    cache, want = make(device, 1, 2, 900)
    q = draw((1, 2, 8, 64), "f32", 2)
    q *= np.float32(10.0) ** np.array([-36, -31, -20, -3, 0, 5, 20, 30], np.float32)[None, None, :, None]
    q[0, 0, 4, 5] = 127.0 * 2.0 ** 4  # the largest of its row, exactly at the edge of a step
    np.testing.assert_array_equal(select(device, cache, (1, 2, 900), q, 5), want.select(q, 5))


def test_select_of_the_largest_products(device):
    """Units of 2^9, and products with them up to FP32's largest number, whose codes take the largest power of two."""
    for tiles in (15, 600):
        k = draw((1, 1, 64 * tiles, 64), "f32", 3, 10000.0)
        k[0, 0, 0] = 49152.0
        cache, want = make(device, 1, 1, 64 * tiles, k=k, v=k)
        assert np.all(want.units == 512.0)
        q = draw((1, 1, 6, 64), "f32", 2)
        largest = np.array([3.4e38, 3.0e38, 1.8e38, 1.6e38, 8e37, 1e37]) / 512
        q *= (largest / np.abs(q[0, 0]).max(-1)).astype(np.float32)[None, None, :, None]
        np.testing.assert_array_equal(select(device, cache, (1, 1, 64 * tiles), q, 5), want.select(q, 5))


@pytest.mark.parametrize("element,layout", [("f32", "heads"), ("f16", "tokens")])
@pytest.mark.parametrize("e,h,n,rows,count", [(1, 8, 1, 1, 1), (1, 8, 640, 3, 4), (2, 3, 1000, 20, 16), (1, 1, 9000, 2, 100),
                                              (1, 2, 777, 300, 3), (1, 8, 640, 600, 70), (1, 2, 640, 300, 300)])
def test_attention_over_listed_blocks(device, e, h, n, rows, count, element, layout):
    """Listed in any order, some twice, some that are no blocks."""
    print(f"{count} listed blocks of {e} x {h} x {n}, {rows} queries, {element} {layout}", flush=True)
    rng = np.random.default_rng(n)
    cache, want = make(device, e, h, n, element, layout, seed=n)
    q = draw((e, h, rows, 64), element, n + 3, 1.5)
    tiles = -(-n // 64)
    blocks = rng.integers(0, tiles, (e, h, rows, count)).astype(np.int32)
    odd = rng.random(blocks.shape)
    blocks[odd < 0.1] = -1
    blocks[odd > 0.95] = tiles
    blocks[odd > 0.97] = 2 ** 31 - 1
    blocks[odd > 0.98] = -2 ** 31
    keep = rng.random((e, n)) < 0.7
    got = attend(device, cache, (e, h, n), q, element, layout, keep=keep, blocks=blocks)
    check(got, want.attend(q, keep=keep, blocks=blocks), element, want)


@pytest.mark.parametrize("e,h,n,rows,count", [(2, 3, 1000, 20, 16), (1, 1, 70000, 40, 1000), (1, 8, 640, 600, 10),
                                              (1, 2, 777, 300, 3)])
def test_fp16_weights_of_listed_blocks_are_pairs(device, e, h, n, rows, count):
    """check()'s bound of FP32 weights (pairs, 2^-21 of the values), and the output's rounding."""
    rng = np.random.default_rng(n)
    cache, want = make(device, e, h, n, "f16", seed=n)
    q = draw((e, h, rows, 64), "f16", n + 3, 1.5)
    blocks = rng.integers(0, -(-n // 64), (e, h, rows, count)).astype(np.int32)
    out, lse = attend(device, cache, (e, h, n), q, "f16", blocks=blocks)
    exact, lse64, magnitude = want.attend(q, blocks=blocks)
    check((out, lse), (exact, lse64, magnitude), "f16", want)
    ds, v = 2.0 ** -17 * magnitude, np.abs(want.v).max()
    bound = v * (4 * ds + 2.0 ** -21 + want.k.shape[2] * (2.0 ** -27 + 2.0 ** -30)) + np.abs(exact) * 2.0 ** -11 + 2.0 ** -25
    off = np.abs(out.astype(np.float64) - exact)
    assert np.all(off <= bound), f"{(off - bound).max():.3e} past the bound"
    # Errors of scores are random and far below that bound; one rounding of the weights would add as much again as the
    # output's own, whose mean square is a twelfth of a step's: of 2,560 outputs or more to some 4%.
    step = np.maximum(2.0 ** (np.floor(np.log2(np.abs(exact) + 1e-300)) - 10), 2.0 ** -24)
    assert np.mean(off ** 2) <= 1.1 * np.mean(step ** 2) / 12


def test_every_block_listed_is_attention_over_all(device):
    e, h, n, rows = 1, 8, 1500, 9
    cache, want = make(device, e, h, n)
    q = draw((e, h, rows, 64), "f32", 2)
    blocks = np.broadcast_to(np.arange(24, dtype=np.int32), (e, h, rows, 24))
    check(attend(device, cache, (e, h, n), q, blocks=blocks), want.attend(q), "f32", want)


# ---- the calls together ----

class Runtime:
    """Streams and graphs of the HIP runtime that the library uses."""

    def __init__(self):
        self.rt = hipmem.runtime()
        self.stream = ctypes.c_void_p()
        self.ok(self.rt.hipStreamCreateWithFlags(ctypes.byref(self.stream), ctypes.c_uint(1)))

    def ok(self, code):
        assert code == 0, f"HIP error {code}"

    def wait(self):
        self.ok(self.rt.hipStreamSynchronize(self.stream))

    def capture(self, fn):
        graph, self.exec = ctypes.c_void_p(), ctypes.c_void_p()
        self.ok(self.rt.hipStreamBeginCapture(self.stream, ctypes.c_int(1)))
        fn()
        self.ok(self.rt.hipStreamEndCapture(self.stream, ctypes.byref(graph)))
        self.ok(self.rt.hipGraphInstantiate(ctypes.byref(self.exec), graph, None, None, ctypes.c_size_t(0)))
        self.ok(self.rt.hipGraphDestroy(graph))

    def launch(self):
        self.ok(self.rt.hipGraphLaunch(self.exec, self.stream))


class Run:
    """Encode, select, attend over the chosen blocks and over all: buffers of one run."""

    def __init__(self, device, e, h, n, rows, count, element, seed):
        self.device, self.shape, self.rows, self.count, self.element = device, (e, h, n), rows, count, element
        dtype = DTYPES[element]
        self.k, self.v, self.q = (hipmem.DeviceArray((e, h, r, 64), dtype) for r in (n, n, rows))
        self.cache = hipmem.DeviceArray((icl4.cache_bytes(self.shape),), np.uint8)
        self.blocks = hipmem.DeviceArray((e, h, rows, count), np.int32)
        self.outs = [hipmem.DeviceArray((e, h, rows, 64), dtype) for _ in range(2)]
        self.lse = [hipmem.DeviceArray((e, h, rows), np.float32) for _ in range(2)]
        self.space = workspace(device, self.shape, rows, count)
        self.dense = workspace(device, self.shape, rows)
        self.fill(seed)

    def fill(self, seed):
        e, h, n = self.shape
        k, v, q = (draw((e, h, r, 64), self.element, seed + i, 1.2) for i, r in enumerate((n, n, self.rows)))
        for d, a in ((self.k, k), (self.v, v), (self.q, q)):
            assert hipmem.runtime().hipMemcpy(d.ptr, a.ctypes.data, d.nbytes, hipmem.H2D) == 0

    def enqueue(self, stream):
        kind = {"element": self.element, "stream": stream}
        icl4.encode(self.device, self.shape, self.k, self.v, self.cache, **kind)
        icl4.select(self.device, self.shape, self.cache, self.q, self.rows, self.count, self.blocks, **self.space, **kind)
        icl4.attention(self.device, self.shape, self.cache, self.q, self.rows, self.outs[0], blocks=self.blocks,
                       n_blocks=self.count, lse=self.lse[0], **self.space, **kind)
        icl4.attention(self.device, self.shape, self.cache, self.q, self.rows, self.outs[1], lse=self.lse[1],
                       **self.dense, **kind)

    def results(self):
        return [a.to_host() for a in (self.blocks, *self.outs, *self.lse)]


@pytest.mark.parametrize("element", ["f32", "f16"])
def test_a_run_is_captured_and_replayed(device, element):
    """The whole run in a graph, replayed on new inputs with eager work between: bitwise the eager results."""
    runtime = Runtime()
    runs = [Run(device, 2, 4, 1300, 70, 5, element, 1), Run(device, 1, 8, 5000, 2, 9, element, 2)]
    eager = [Run(device, 2, 4, 1300, 70, 5, element, 1), Run(device, 1, 8, 5000, 2, 9, element, 2)]
    for run, other in zip(runs, eager):
        runtime.capture(lambda: run.enqueue(runtime.stream.value))
        for replay in range(4):
            print(f"replay {replay}", flush=True)
            run.fill(10 * replay), other.fill(10 * replay)
            hipmem.synchronize()
            runtime.launch()
            runtime.wait()
            got = run.results()
            other.enqueue(None)
            hipmem.synchronize()
            for a, b in zip(got, other.results()):
                np.testing.assert_array_equal(a, b)
        want = icl4_np.Cache(run.k.to_host(), run.v.to_host())
        q = run.q.to_host()
        np.testing.assert_array_equal(got[0], want.select(q, run.count))
        check((got[1], got[3]), want.attend(q, blocks=got[0]), element, want)
        check((got[2], got[4]), want.attend(q), element, want)


def test_two_streams_at_once(device):
    """Runs on two streams with workspaces of their own: each bitwise its run alone."""
    streams = [Runtime(), Runtime()]
    runs = [Run(device, 1, 8, 4000, 40, 6, "f32", 1), Run(device, 1, 8, 6000, 1, 20, "f32", 2)]
    alone = []
    for run in runs:
        run.enqueue(None)
        hipmem.synchronize()
        alone.append(run.results())
    for _ in range(5):
        for stream, run in zip(streams, runs):
            run.enqueue(stream.stream.value)
    for stream in streams:
        stream.wait()
    for run, want in zip(runs, alone):
        for a, b in zip(run.results(), want):
            np.testing.assert_array_equal(a, b)


def test_shared_sources_and_a_cache_past_32_bits(device):
    """One estimator's rows shared by 64 pairs (strides of 0): a 4.8 GB cache whose last pair answers as its first."""
    e, h, n = 8, 8, 1_060_000
    rng = np.random.default_rng(0)
    k, v = (put(rng.standard_normal((n, 64), dtype=np.float32).astype(np.float16)) for _ in range(2))
    cache = hipmem.DeviceArray((icl4.cache_bytes((e, h, n)),), np.uint8)
    assert cache.nbytes > 2 ** 32
    icl4.encode(device, (e, h, n), k, v, cache, element="f16", k_strides=(0, 0, 64), v_strides=(0, 0, 64))
    q = put(rng.standard_normal((1, 64), dtype=np.float32).astype(np.float16))
    out, lse = hipmem.DeviceArray((e, h, 1, 64), np.float16), hipmem.DeviceArray((e, h, 1), np.float32)
    blocks = hipmem.DeviceArray((e, h, 1, 30), np.int32)
    space = workspace(device, (e, h, n), 1, 30)
    dense = workspace(device, (e, h, n), 1)
    icl4.attention(device, (e, h, n), cache, q, 1, out, element="f16", q_strides=(0, 0, 0), lse=lse, **dense)
    icl4.select(device, (e, h, n), cache, q, 1, 30, blocks, element="f16", q_strides=(0, 0, 0), **space)
    hipmem.synchronize()
    a, s, b = out.to_host().reshape(64, 64), lse.to_host().ravel(), blocks.to_host().reshape(64, 30)
    assert np.all(a == a[0]) and np.all(s == s[0]) and np.all(b == b[0]) and np.all(np.diff(b[0]) > 0)
    # log of the sum over n keys of exp(s), s of mean 0: log n at least, and finite.
    assert np.log(n) - 0.1 < s[0] < np.log(n) + 40
    icl4.attention(device, (e, h, n), cache, q, 1, out, element="f16", q_strides=(0, 0, 0), lse=lse, blocks=blocks,
                   n_blocks=30, **space)
    hipmem.synchronize()
    a, s = out.to_host().reshape(64, 64), lse.to_host().ravel()
    assert np.all(a == a[0]) and np.all(s == s[0])


def test_small_workspaces_are_refused(device):
    cache, _ = make(device, 1, 8, 5000)
    q = put(draw((1, 8, 1, 64), "f32", 1))
    out = hipmem.DeviceArray((1, 8, 1, 64))
    need = icl4.workspace_bytes(device, (1, 8, 5000), 1)
    assert need > 0
    space = hipmem.DeviceArray((need,), np.uint8)
    for kw in ({}, {"workspace": space, "workspace_bytes": need - 1}, {"workspace": None, "workspace_bytes": need}):
        with pytest.raises(hip.HipError, match="workspace must hold") as info:
            icl4.attention(device, (1, 8, 5000), cache, q, 1, out, **kw)
        assert info.value.status == hip.INVALID_ARGUMENT
    blocks = hipmem.DeviceArray((1, 8, 200, 4), np.int32)
    with pytest.raises(hip.HipError, match="workspace must hold"):  # its scores do not fit one launch
        icl4.select(device, (1, 8, 70000), cache, q, 200, 4, blocks)
    with pytest.raises(hip.HipError, match="too many queries"):
        icl4.select(device, (8190, 8, 64), cache, q, 30000, 4, blocks)
    with pytest.raises(hip.HipError, match="too many queries"):
        icl4.attention(device, (8190, 8, 64), cache, q, 30000, out, out_strides=(30000 * 512, 64, 512))
