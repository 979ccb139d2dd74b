"""Attention for training, its backward pass and dropout on the GPU against their definitions in float64 (training_np.py),
within bounds worked out beforehand.

Bounds, relative to the sums of magnitudes that the oracle takes beside each result. A score is a sum of 64 products. FP32
operands are pairs of FP16 values: a half step of a half step, 2^-22, each, and the product of the two lower, 2^-22, left
out; 16-bit operands are whole. Their FP32 sums are off by 2^-18 at most (24 additions of sums inside the matrix cores), the
scale by less. So with A the largest sum of |scale q k| the score is off by ds <= 2^-17 A, and a weight by 2 ds, relative.
FP32 sums over N rows (16 in one addition) are off by N 2^-27, weights and dS by their rounding, with the left-out product
and the other operand's: rp = (2^-20, 2^-11, 2^-8: half a step of 16-bit types) for (FP32, FP16, BF16), an exponential by
2^-22. An output's own rounding is half a step, h = (2^-24, 2^-11, 2^-8).

  out:  out_abs (2 ds + rp + N 2^-26 + 2^-20) + h |out|
  dv:   dv_abs (2 ds + rp + Q 2^-26 + 2^-20) + h |dv|
  dS:   its dP is a product like a score's, 2^-18 + rp of its magnitude; its delta is off by what out is, and by 2^-20 of
        its own magnitude: dS_abs (2 ds + rp + 2^-17 + [out's bound and h])
  dq:   dq_abs ([dS's] + rp + N 2^-26 + 2^-20) + h |dq|; dk the same with Q.

FP16 values below 2^-14 are off by 2^-25. FP32's and FP16's weights (and dS) come by a power with which the largest of them
times its tile's power is 2^13 at least, and FP32's rows by one with which the largest number of the tile's turn is 2^14 at
least, its other rows within 2^14 of it: every term may miss 2^-37 (2^-25 2^15 / 2^13 / 2^14) of the largest factor times
its turn's largest number, which is at most 2^14 that row's own, and at most the largest of all. A row's own small numbers
miss 2^-25 / 2^14 of the turn's largest: as much again. And values 2^40 below the largest of their context keep 2^-79 of it.

FP16 results below its normal numbers round by 2^-25. A key's sums take every head of its group: Q stands for all of them."""

import ctypes

import numpy as np
import pytest

import training_np
from ironicl_amd import hip, hipmem, training

pytestmark = pytest.mark.gpu
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
PARTS = {"f32": 2.0 ** -20, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
SCORE = 2.0 ** -17
# Weights below 2^-126 are taken as 0, and parts of products' operands below that: a result of 2^15 terms with operands up to
# 2^11 misses 2^-126 2^15 2^11 at most.
TINY = {"f32": 2.0 ** -100, "f16": 2.0 ** -25, "bf16": 2.0 ** -100}
SEED = 0x9A3B5C7D12345678


@pytest.fixture(scope="module")
def device():
    return hip.Device(0)


def encode(x, element):
    """float64 as the element's bits, to nearest, ties to even."""
    if element == "f32":
        return np.asarray(x, np.float32)
    if element == "f16":
        return np.asarray(x, np.float16)
    b = np.asarray(x, np.float32).view(np.uint32)
    rounded = (b + 0x7FFF + (b >> 16 & 1) >> 16).astype(np.uint16)
    return np.where(np.isnan(np.asarray(x, np.float32)), np.uint16(0x7FC0), rounded)


def decode(a, element):
    if element == "bf16":
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


def put(a):
    return None if a is None else hipmem.DeviceArray.from_host(np.ascontiguousarray(a))


MARK = 77.0  # in every number of a tensor that a call may leave


class Tensor:
    """[E, H, N, 64] on the device, head-major or as token rows [E, N, H * 64 + gap]; `host` float64, rounded to the element."""

    def __init__(self, shape, element, layout="heads", host=None):
        e, h, n, _ = shape
        self.shape, self.layout, self.element = shape, layout, element
        width = h * 64 + 16
        self.strides, full = ((h * n * 64, n * 64, 64), (e, h, n, 64)) if layout == "heads" else ((n * width, 64, width), (e, n, width))
        bits = encode(np.full(full, MARK), element)
        if host is not None:
            self.view(bits)[:] = encode(host, element)
        self.array = put(bits)
        self.values = None if host is None else decode(encode(host, element), element)

    def view(self, a):
        if self.layout == "heads":
            return a
        e, h, n, _ = self.shape
        return np.lib.stride_tricks.as_strided(a, self.shape, [s * a.itemsize for s in self.strides] + [a.itemsize])

    def get(self):
        a = self.array.to_host()
        if self.layout != "heads":
            assert np.all(decode(a[:, :, self.shape[1] * 64:], self.element) == MARK), "written past the heads"
        return decode(self.view(a), self.element)


def normal(shape, seed, scale=1.0):
    return np.random.default_rng(seed).standard_normal(shape) * scale


def workspace(device, shape, element, backward):
    size = training.workspace_bytes(device, shape, element=element, backward=backward)
    # Full of NaN: nothing may hang on what it held.
    return {"workspace": put(np.full(max(size, 16), 255, np.uint8)), "workspace_bytes": size}


class Case:
    """Inputs on the device, the calls on them, and the oracle."""

    def __init__(self, device, e, h, g, m, n, element="f32", layout="heads", q_lengths=None, lengths=None, keep=None,
                 dropped=0, site=3, scale=0.125, seed=0, q=None, k=None, v=None, dout=None):
        self.device, self.shape, self.element, self.layout = device, (e, h, g, m, n), element, layout
        q = normal((e, h, m, 64), seed, 1.3) if q is None else q
        k = normal((e, g, n, 64), seed + 1, 1.1) if k is None else k
        v = normal((e, g, n, 64), seed + 2) if v is None else v
        dout = normal((e, h, m, 64), seed + 3, 0.02) if dout is None else dout
        self.q, self.k, self.v, self.dout = (Tensor(x.shape, element, layout, x) for x in (q, k, v, dout))
        self.q_lengths, self.lengths, self.keep, self.dropped = q_lengths, lengths, keep, dropped
        self.kept = [put(None if x is None else np.asarray(x, np.uint32)) for x in (q_lengths, lengths)]
        self.kept += [put(None if keep is None else training_np.bits(keep)), put(np.array([SEED], np.uint64))]
        self.kind = {"element": element, "scale": scale, "q_strides": self.q.strides, "k_strides": self.k.strides,
                     "v_strides": self.v.strides, "query_lengths": self.kept[0], "lengths": self.kept[1],
                     "keep": self.kept[2], "seed": self.kept[3], "site": site, "dropped": dropped}
        self.space = [workspace(device, self.shape, element, b) for b in (False, True)]
        self.out = Tensor(q.shape, element, layout)
        self.stats = put(np.full((e, h, m, 2), MARK, np.float32))
        self.lse = put(np.full((e, h, m), MARK, np.float32))
        self.grads = [Tensor(x.shape, element, layout) for x in (q, k, v)]
        self.args = (scale, q_lengths, lengths, keep, SEED, site, dropped)

    def forward(self, stream=None):
        training.attention(self.device, self.shape, self.q.array, self.k.array, self.v.array, self.out.array,
                           out_strides=self.out.strides, stats=self.stats, lse=self.lse, stream=stream, **self.kind, **self.space[0])

    def backward(self, stream=None, queries=True, keys=True):
        dq, dk, dv = self.grads
        sides = {"dq": dq.array if queries else None, "dk": dk.array if keys else None, "dv": dv.array if keys else None}
        training.attention_backward(self.device, self.shape, self.q.array, self.k.array, self.v.array, self.out.array,
                                    self.stats, self.dout.array, out_strides=self.out.strides,
                                    dout_strides=self.dout.strides, dq_strides=dq.strides, dk_strides=dk.strides,
                                    dv_strides=dv.strides, stream=stream, **sides, **self.kind, **self.space[1])

    def oracle(self):
        values = [np.nan_to_num(t.values, nan=0.0, posinf=0.0, neginf=0.0) for t in (self.q, self.k, self.v, self.dout)]
        return training_np.Attention(*values[:3], *self.args, dout=values[3])

    def results(self):
        return [self.out.get(), self.lse.to_host(), self.stats.to_host()] + [t.get() for t in self.grads]

    def run(self):
        self.forward()
        self.backward()
        hipmem.synchronize()
        return self.results()

    def check(self, got, queries=True, keys=True):
        want, el = self.oracle(), self.element
        out, lse, stats, dq, dk, dv = got
        n, group = self.shape[4], self.shape[1] // self.shape[2]
        m = self.shape[3] * group
        ds = SCORE * want.magnitude.max(initial=0.0)
        rows = want.inside[:, None, :, None] & np.ones(out.shape, bool)
        held = want.held[:, None, :, None] & np.ones(dk.shape, bool)
        within(out, want.out, want.out_abs * (2 * ds + PARTS[el] + n * 2.0 ** -26 + 2.0 ** -20)
               + floor(want.out_term, n, el) + n * 2.0 ** -79 * np.abs(self.v.values[np.isfinite(self.v.values)]).max(), rows, el, "out")
        empty = np.isneginf(want.lse)
        inside = want.inside[:, None, :] & np.ones(lse.shape, bool)
        assert np.array_equal(np.isneginf(lse) & inside, empty & inside), "queries that attend to nothing"
        assert np.all(stats[inside & empty] == 0) and np.all(out[(inside & empty)] == 0)
        assert np.all(lse[~inside] == MARK) and np.all(stats[~inside] == MARK), "past the queries"
        full = inside & ~empty
        # The same sums under a reference that may be the next whole number.
        total = stats[..., 1].astype(np.float64) * np.exp2(np.where(full, stats[..., 0] - want.r, 0.0))
        assert np.all(stats[full][..., 0] == np.round(stats[full][..., 0]))
        bound = 2 * ds + n * 2.0 ** -26 + 2.0 ** -20
        assert np.all(np.abs(total - want.s)[full] <= bound * want.s[full])
        off = np.abs(lse[full] - want.lse[full]) - (2 * ds + n * 2.0 ** -26 + 2.0 ** -21 * np.abs(want.lse[full]) + 1e-6)
        assert not full.any() or off.max() <= 0, f"lse {off.max():.3e} past the bound"
        forward = 2 * ds + PARTS[el] + n * 2.0 ** -26 + 2.0 ** -20
        score = 2 * ds + PARTS[el] + 2.0 ** -17 + forward + HALF[el] + 2.0 ** -20
        if queries:
            within(dq, want.dq, want.dq_abs * (score + PARTS[el] + n * 2.0 ** -26 + 2.0 ** -20) + floor(want.dq_term, n, el), rows, el, "dq")
        if keys:
            within(dk, want.dk, want.dk_abs * (score + PARTS[el] + m * 2.0 ** -26 + 2.0 ** -20) + floor(want.dk_term, m, el), held, el, "dk")
            within(dv, want.dv, want.dv_abs * (2 * ds + PARTS[el] + m * 2.0 ** -26 + 2.0 ** -20) + floor(want.dv_term, m, el), held, el, "dv")
            masked = held & ~want.attended[:, None, :, None]
            assert np.all(dk[masked] == 0) and np.all(dv[masked] == 0), "gradients of rows that are not attended"


def within(got, want, bound, written, element, name):
    assert np.all(got[~written] == MARK), f"{name}: written past the lengths"
    bound = bound + HALF[element] * np.abs(want) + TINY[element]
    with np.errstate(invalid="ignore"):
        bad = written & ~(np.abs(got - want) <= bound)
    off = np.abs(got - want)[bad]
    where = np.argwhere(bad)[:4].tolist()
    assert not bad.any(), f"{name}: {bad.sum()} of {bad.size} past the bound, by {np.max(off - bound[bad]):.3e}, at {where}"


def floor(term, count, element):
    """What `count` terms may miss: see above."""
    return 0.0 if element == "bf16" else 2 * count * 2.0 ** -37 * np.minimum(term[0] * 2.0 ** 14, term[1])


def random_keep(e, n, seed):
    keep = np.random.default_rng(seed).random((e, n)) < 0.8
    for start in range(0, n, 150):  # whole blocks left out, too
        keep[:, start:start + 70] &= np.random.default_rng(seed + start).random((e, 1)) < 0.6
    return keep


SHAPES = [(1, 8, 8, 1, 1), (1, 8, 8, 3, 63), (2, 4, 4, 16, 64), (1, 8, 2, 17, 65), (1, 3, 3, 1, 1000), (2, 8, 8, 33, 777),
          (1, 8, 1, 65, 2049), (1, 2, 2, 130, 640), (1, 1, 1, 300, 5000), (1, 2, 1, 700, 3), (2, 6, 3, 129, 128),
          (1, 1, 1, 2500, 200), (1, 1, 1, 5, 20011)]


@pytest.mark.parametrize("element,layout", [("f32", "heads"), ("f16", "tokens"), ("bf16", "tokens"), ("f32", "tokens"), ("bf16", "heads")])
@pytest.mark.parametrize("shape", SHAPES)
def test_attention_and_its_gradients(device, shape, element, layout):
    print(f"attention {shape} {element} {layout}", flush=True)
    case = Case(device, *shape, element, layout, seed=shape[4])
    case.check(case.run())


@pytest.mark.parametrize("element", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("shape", [(1, 8, 2, 1, 9000), (2, 8, 1, 1, 8200), (1, 4, 2, 2, 8193), (1, 6, 2, 2, 10000), (2, 2, 2, 2, 9001),
                                   (1, 8, 8, 4, 20000), (1, 2, 1, 8, 9000), (3, 5, 5, 1, 130)])
def test_few_rows(device, shape, element):
    """Single queries of heads that share keys, and a few of them, over long contexts, uneven, masked, with dropout."""
    print(f"few rows {shape} {element}", flush=True)
    e, h, g, m, n = shape
    for uneven, dropped in ((False, 0), (True, 9000)):
        lengths = np.array([n, n // 2, 0])[:e] if uneven else None
        q_lengths = np.array([max(1, m - 1), m, m])[:e] if uneven else None
        case = Case(device, *shape, element, "tokens", q_lengths, lengths, random_keep(e, n, 4) if uneven else None, dropped, seed=n)
        case.check(case.run())


@pytest.mark.parametrize("element,layout", [("f32", "heads"), ("f16", "heads"), ("bf16", "tokens")])
@pytest.mark.parametrize("dropped", [1, 6554, 40000, 65535])
@pytest.mark.parametrize("shape", [(1, 2, 2, 1, 77), (2, 4, 2, 70, 200), (1, 1, 1, 200, 1300), (1, 2, 1, 600, 37)])
def test_dropout_of_the_weights(device, shape, dropped, element, layout):
    print(f"attention {shape} {element} {layout}, {dropped} dropped", flush=True)
    case = Case(device, *shape, element, layout, dropped=dropped, seed=dropped)
    case.check(case.run())


@pytest.mark.parametrize("element,layout", [("f32", "tokens"), ("f16", "tokens"), ("bf16", "heads")])
@pytest.mark.parametrize("e,h,g,m,n,q_lengths,lengths,masked", [
    (3, 4, 2, 40, 200, (40, 7, 0), (200, 129, 64), False),
    (3, 4, 4, 40, 200, None, (0, 200, 1), True),
    (2, 2, 1, 150, 1000, (150, 33), (1000, 500), True),
    (2, 2, 2, 5, 700, (4000000000, 1), (4000000000, 65), True),
    (1, 1, 1, 300, 64, (1,), None, True),
    (1, 8, 8, 1, 3000, None, None, True),
    (4, 2, 2, 257, 70, (257, 256, 1, 0), (70, 0, 64, 65), True),
])
def test_lengths_and_masks(device, e, h, g, m, n, q_lengths, lengths, masked, element, layout):
    print(f"attention {(e, h, g, m, n)} {q_lengths} {lengths} {masked} {element} {layout}", flush=True)
    keep = random_keep(e, n, n) if masked else None
    for dropped in (0, 20000):
        case = Case(device, e, h, g, m, n, element, layout, q_lengths, lengths, keep, dropped, seed=n + m)
        case.check(case.run())


@pytest.mark.parametrize("element", ["f32", "f16", "bf16"])
def test_what_is_not_attended_does_not_matter(device, element):
    """NaN, infinities and the largest numbers in rows that are masked out, past the lengths and in queries past theirs, and
    an estimator whose mask leaves no row."""
    keep = random_keep(3, 200, 5)
    keep[2] = False
    q, k, v, dout = normal((3, 2, 50, 64), 1), normal((3, 2, 200, 64), 2), normal((3, 2, 200, 64), 3), normal((3, 2, 50, 64), 4)
    lengths, q_lengths = np.array([200, 130, 200]), np.array([50, 20, 50])
    attended = keep & (np.arange(200) < lengths[:, None])
    for x in (k, v):
        for i, bad in enumerate((np.nan, np.inf, -np.inf, 3e38 if element != "f16" else 65504.0)):
            x[..., i::8] = np.where(attended[:, None, :, None], x[..., i::8], bad)
    late = (np.arange(50) >= q_lengths[:, None])[:, None, :, None]
    q, dout = np.where(late, np.nan, q), np.where(late, np.inf, dout)
    # What the empty estimator's queries and their gradient hold does not reach any result either.
    q[2, :, 3], dout[2, :, 4] = np.nan, np.inf
    for dropped in (0, 9999):
        case = Case(device, 3, 2, 2, 50, 200, element, "heads", q_lengths, lengths, keep, dropped, q=q, k=k, v=v, dout=dout)
        case.check(case.run())


@pytest.mark.parametrize("element", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("size", [30.0, 1000.0, 16384.0, 131072.0])
def test_large_scores(device, element, size):
    """Scores up to 2^18: whole numbers, exact in every form, so that a weight is off by its exponential alone and near ties
    keep their weights."""
    if element == "f16" and size > 2.0 ** 15:
        pytest.skip("queries past FP16's range")
    rng = np.random.default_rng(8)
    k = rng.integers(-2, 3, (1, 2, 300, 64)).astype(float)
    q = rng.integers(-2, 3, (1, 2, 40, 64)) * size
    case = Case(device, 1, 2, 2, 40, 300, element, q=q, k=k, scale=2.0 ** -7)
    got, want = case.run(), case.oracle()
    # log2(e) scale is rounded to 2^-25, and its product with a score to 2^-24 of itself.
    ds = 2.0 ** -23 * want.magnitude.max()
    n = 300
    rest = 6 * ds + 4 * PARTS[element] + HALF[element] + n * 2.0 ** -25 + 2.0 ** -16
    weights = 4 * ds + 2 * PARTS[element] + n * 2.0 ** -26 + 2.0 ** -20
    for name, have, exact, bound, term, count in (
            ("out", got[0], want.out, want.out_abs * weights, want.out_term, n), ("dq", got[3], want.dq, want.dq_abs * rest, want.dq_term, n),
            ("dk", got[4], want.dk, want.dk_abs * rest, want.dk_term, 40), ("dv", got[5], want.dv, want.dv_abs * weights, want.dv_term, 40)):
        within(have, exact, bound + floor(term, count, element), np.ones(have.shape, bool), element, name)


@pytest.mark.parametrize("exponent", [-90, -40, 40, 90])
def test_fp32_gradients_of_any_size(device, exponent):
    """Powers of two pass through: dq, dk and dv are the same numbers, scaled, bit for bit, as long as no part of dout
    (2^-6) or of dS (2^-6 times a weight, down to 2^-24 of it) falls below 2^-126. At 2^-90 some do: each of 130 terms may
    miss 2^-126 times an operand up to 8, and a sum that misses one may round the other way once in each of its additions,
    fewer than 64, by 2^-24 of a sum of magnitudes."""
    a = Case(device, 1, 2, 2, 70, 130, dropped=3000, seed=4)
    dout = a.dout.values
    b = Case(device, 1, 2, 2, 70, 130, dropped=3000, seed=4, dout=dout * 2.0 ** exponent)
    want = a.oracle()
    for x, y, size in zip(a.run()[3:], b.run()[3:], (want.dq_abs, want.dk_abs, want.dv_abs)):
        if exponent < -80:
            assert np.all(np.abs(x * 2.0 ** exponent - y) <= size * 2.0 ** (exponent - 18) + 130 * 8 * 2.0 ** -126)
        else:
            np.testing.assert_array_equal(x * 2.0 ** exponent, y)


def spread(shape, seed, low, high):
    """Normal numbers, every row times a power of two of its own."""
    x = normal(shape, seed)
    return x * 2.0 ** np.random.default_rng(seed + 99).integers(low, high + 1, shape[:3])[..., None]


@pytest.mark.parametrize("element", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("which", ["values", "gradients", "scores", "all", "zeros", "channel"])
def test_rows_of_very_different_sizes(device, which, element):
    """Rows side by side whose sizes span up to 60 binades (FP16's own range for FP16), rows of zeros, and one channel that
    outweighs the others: every result is within the same bounds of its own terms' sizes."""
    e, h, g, m, n = 2, 2, 1, 90, 300
    wide = (-30, 30) if element != "f16" else (-6, 6)
    q, k, v, dout = normal((e, h, m, 64), 1), normal((e, g, n, 64), 2), normal((e, g, n, 64), 3), normal((e, h, m, 64), 4)
    if which in ("values", "all"):
        v = spread(v.shape, 5, *wide)
    if which in ("gradients", "all"):
        dout = spread(dout.shape, 6, *wide)
    if which in ("scores", "all"):
        q, k = spread(q.shape, 7, wide[0] // 2, 1), spread(k.shape, 8, wide[0] // 2, 1)
    if which == "zeros":
        for x in (q, k, v, dout):
            x[:, :, ::3] = 0.0
        k[:, :, 64:128], v[:, :, 64:128], v[1], dout[:, :, 64:] = 0.0, 0.0, 0.0, 0.0
    if which == "channel":
        k[..., 5] *= 50.0
        v[..., 9] *= 300.0
        dout[..., 11] *= 1000.0
    for dropped in (0, 9000):
        case = Case(device, e, h, g, m, n, element, "tokens", dropped=dropped, q=q, k=k, v=v, dout=dout, keep=random_keep(e, n, 3))
        case.check(case.run())


@pytest.mark.parametrize("element", ["f32", "bf16"])
def test_one_side_alone(device, element):
    keep = random_keep(2, 333, 1)
    for queries, keys in ((True, False), (False, True)):
        case = Case(device, 2, 4, 2, 90, 333, element, "tokens", (90, 44), (333, 100), keep, 5000)
        case.forward()
        case.backward(queries=queries, keys=keys)
        hipmem.synchronize()
        got = case.results()
        case.check(got, queries, keys)
        for t in got[3:4] if keys else got[4:]:
            assert np.all(t == MARK)


@pytest.mark.parametrize("element", ["f32", "f16", "bf16"])
def test_the_same_call_gives_the_same_bits(device, element):
    case = Case(device, 1, 8, 2, 100, 5000, element, dropped=6554)
    first = case.run()
    for x, y in zip(first, case.run()):
        np.testing.assert_array_equal(x, y)


@pytest.mark.parametrize("dropped", [0, 6554])
@pytest.mark.parametrize("element", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("number", [np.inf, -np.inf, np.nan])
def test_gradients_that_are_not_finite(device, number, element, dropped):
    """One such number of the output's gradient: it shows in its query's gradient and in every key's, as a step that scales
    its loss looks for, and other queries' stay: FP32's and FP16's powers may differ, by which 200 terms miss 2^-37 each."""
    e, h, m, n = 1, 2, 70, 200
    first = Case(device, e, h, h, m, n, element, dropped=dropped)
    clean = first.run()
    dout = first.dout.values.copy()
    dout[0, 1, 41, 7] = number
    got = Case(device, e, h, h, m, n, element, dropped=dropped, dout=dout).run()
    dq, dk, dv = got[3:]
    assert not np.isfinite(dq[0, 1, 41]).any()
    assert not np.isfinite(dk[0, 1]).any() and not np.isfinite(dv[0, 1, :, 7]).any()
    assert np.isfinite(dk[0, 0]).all() and np.isfinite(dv[0, 0]).all()
    dq[0, 1, 41] = clean[3][0, 1, 41]
    assert np.all(np.abs(dq - clean[3]) <= 2 * HALF[element] * np.abs(dq) + 2.0 ** -20 * np.abs(dq).max())
    for x, y in zip(got[:3], clean[:3]):
        np.testing.assert_array_equal(x, y)


@pytest.mark.parametrize("element", ["f32", "bf16"])
def test_two_calls_at_once(device, element):
    """On two streams, with a workspace each: the results of one after the other."""
    cases = [Case(device, 1, 4, 2, 200, 6000, element, dropped=6554), Case(device, 2, 4, 4, 33, 1500, element)]
    alone = [case.run() for case in cases]
    rt = hipmem.runtime()
    streams = [ctypes.c_void_p(), ctypes.c_void_p()]
    for s in streams:
        assert rt.hipStreamCreate(ctypes.byref(s)) == 0
    for _ in range(4):
        for call in ("forward", "backward"):
            for case, s in zip(cases, streams):
                getattr(case, call)(s.value)
    hipmem.synchronize()
    for case, want in zip(cases, alone):
        for x, y in zip(case.results(), want):
            np.testing.assert_array_equal(x, y)
    for s in streams:
        assert rt.hipStreamDestroy(s) == 0


def test_the_most_pairs(device):
    """65,535 estimators of one head, of two queries and three rows."""
    rng = np.random.default_rng(0)
    e = 65535
    lengths, keep = rng.integers(0, 4, e), rng.random((e, 3)) < 0.7
    case = Case(device, e, 1, 1, 2, 3, "f32", "heads", rng.integers(0, 3, e), lengths, keep, 9000)
    case.check(case.run())


def test_the_most_rows(device):
    """2^24 rows of keys that are 0: every weight is the same, and values of row number mod 16 have whole sums."""
    n, e, h, m = 1 << 24, 1, 1, 3
    shape = (e, h, h, m, n)
    k = put(np.zeros(n * 64, np.uint16))
    v = put(np.tile(np.repeat(np.arange(16, dtype=np.float16), 64).view(np.uint16), n // 16))
    q = put(encode(normal((e, h, m, 64), 1), "f16"))
    out, stats, lse = put(np.zeros((m, 64), np.float16)), put(np.zeros((m, 2), np.float32)), put(np.zeros(m, np.float32))
    training.attention(device, shape, q, k, v, out, element="f16", stats=stats, lse=lse, **workspace(device, shape, "f16", False))
    dout = put(np.full((m, 64), 16.0, np.float16))
    dq = put(np.full((m, 64), 1, np.float16))
    dk, dv = hipmem.DeviceArray((n * 64,), np.uint16), hipmem.DeviceArray((n * 64,), np.uint16)
    training.attention_backward(device, shape, q, k, v, out, stats, dout, dq=dq, dk=dk, dv=dv, element="f16",
                                **workspace(device, shape, "f16", True))
    hipmem.synchronize()
    assert np.all(out.to_host() == 7.5) and np.all(stats.to_host() == [0, n])
    np.testing.assert_allclose(lse.to_host(), np.log(n), rtol=2.0 ** -22)
    assert np.all(dq.to_host() == 0)  # the keys are 0
    # 3 * 16 / 2^24 for every number of dv.
    assert np.all(dv.to_host().view(np.float16) == np.float16(48.0 / n))


def test_shared_inputs_have_gradients_of_their_own(device):
    """Keys and values with strides of 0 over heads and estimators."""
    k, v = normal((1, 1, 150, 64), 1), normal((1, 1, 150, 64), 2)
    wide = Case(device, 2, 3, 3, 20, 150, k=np.broadcast_to(k, (2, 3, 150, 64)).copy(), v=np.broadcast_to(v, (2, 3, 150, 64)).copy())
    case = Case(device, 2, 3, 3, 20, 150)
    case.k, case.v = Tensor(k.shape, "f32", "heads", k), Tensor(v.shape, "f32", "heads", v)
    case.kind["k_strides"] = case.kind["v_strides"] = (0, 0, 64)
    for x, y in zip(case.run(), wide.run()):
        np.testing.assert_array_equal(x, y)


def test_gradients_against_differences(device):
    """The loss sum(out * dout) at q, k, v moved a step either way along a random direction."""
    args = dict(dropped=12000, seed=21)
    case = Case(device, 1, 2, 1, 9, 40, **args)
    grads = case.run()[3:]
    values = [t.values for t in (case.q, case.k, case.v)]
    for i, name in enumerate("qkv"):
        step = normal(values[i].shape, 50 + i, 2.0 ** -6)
        loss = []
        for sign in (1.0, -1.0):
            moved = dict(zip("qkv", values), **{name: values[i] + sign * step}, dout=case.dout.values)
            want = training_np.Attention(moved["q"], moved["k"], moved["v"], *case.args)
            loss.append((want.out * case.dout.values).sum())
        # Central differences in float64 are off by the third derivative: 2^-12 of the first order, and then some.
        assert abs((loss[0] - loss[1]) / 2 - (grads[i] * step).sum()) <= 2.0 ** -8 * np.abs(grads[i] * step).sum()


def test_offsets_past_32_bits(device):
    """Rows 2^22 elements apart: the last start past 2^32 bytes and past 2^31 elements."""
    e, h, m, n, pitch = 1, 1, 3, 520, 1 << 22
    k, v = normal((e, h, n, 64), 1), normal((e, h, n, 64), 2)
    case = Case(device, e, h, h, m, n, "bf16", k=k, v=v)
    want = case.run()
    far = hipmem.DeviceArray(((n - 1) * pitch + 256,), np.uint16)  # k in columns 0 .. 63, v, dk and dv after it
    rt = hipmem.runtime()
    rt.hipMemcpy2D.argtypes = [ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_size_t, ctypes.c_size_t, ctypes.c_int]
    for i, t in enumerate((case.k, case.v)):
        assert rt.hipMemcpy2D(far.ptr + 128 * i, 2 * pitch, t.array.ptr, 128, 128, n, hipmem.D2D) == 0
    strides = (0, 0, pitch)
    case.kind["k_strides"] = case.kind["v_strides"] = strides
    kind = dict(case.kind, **case.space[0])
    training.attention(device, case.shape, case.q.array, far.ptr, far.ptr + 128, case.out.array, out_strides=case.out.strides,
                       stats=case.stats, lse=case.lse, **kind)
    kind = dict(case.kind, **case.space[1])
    training.attention_backward(device, case.shape, case.q.array, far.ptr, far.ptr + 128, case.out.array, case.stats,
                                case.dout.array, dq=case.grads[0].array, dk=far.ptr + 256, dv=far.ptr + 384,
                                dk_strides=strides, dv_strides=strides, **kind)
    for i, t in enumerate(case.grads[1:]):
        assert rt.hipMemcpy2D(t.array.ptr, 128, far.ptr + 256 + 128 * i, 2 * pitch, 128, n, hipmem.D2D) == 0
    hipmem.synchronize()
    for x, y in zip(case.results(), want):
        np.testing.assert_array_equal(x, y)


# ---- dropout ----

@pytest.mark.parametrize("element", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,width,gap", [(1, 1, 0), (1, 7, 0), (3, 8, 0), (5, 13, 8), (100, 512, 0), (33, 1000, 16), (2049, 96, 0), (700, 1, 8)])
@pytest.mark.parametrize("dropped", [0, 1, 6554, 65535])
def test_dropout(device, rows, width, gap, dropped, element):
    """One FP32 product and one addition: half a step of each, and of the result's rounding."""
    print(f"dropout {rows} x {width} {element} {dropped}", flush=True)
    pitch = -(-width // 8) * 8 + gap
    x, residual = (encode(normal((rows, pitch), i), element) for i in (1, 2))
    seed = put(np.array([SEED], np.uint64))
    kept = training_np.kept_numbers(SEED, 5, dropped, rows, width) * (65536.0 / (65536 - dropped))
    for second in (None, residual):
        for place in ("apart", "x", "residual"):
            if place == "residual" and second is None:
                continue
            dx, dr, out = put(x), put(second), put(encode(np.full((rows, pitch), MARK), element))
            to, held = {"apart": (out, encode(np.full((rows, pitch), MARK), element)), "x": (dx, x), "residual": (dr, residual)}[place]
            training.dropout(device, rows, width, dx, to, element=element, residual=dr, x_stride=pitch, residual_stride=pitch,
                             out_stride=pitch, seed=seed, site=5, dropped=dropped)
            hipmem.synchronize()
            got = to.to_host()
            term = decode(x, element)[:, :width] * kept
            want = term + (decode(second, element)[:, :width] if second is not None else 0.0)
            bound = 2.0 ** -23 * np.abs(term) + (2.0 ** -24 + HALF[element]) * np.abs(want) + TINY[element]
            assert np.all(np.abs(decode(got, element)[:, :width] - want) <= bound)
            np.testing.assert_array_equal(got[:, width:], held[:, width:])


def test_dropout_is_its_own_gradient(device):
    """D is diagonal: sum(y D(x)) = sum(x D(y)), and with nothing dropped the result is x."""
    x, y = (np.random.default_rng(i).integers(-8, 9, (40, 70)).astype(np.float32) for i in (1, 2))
    x, y = (np.pad(a, ((0, 0), (0, 2))) for a in (x, y))
    seed, outs = put(np.array([SEED], np.uint64)), []
    for a in (x, y):
        out = put(np.zeros((40, 72), np.float32))
        training.dropout(device, 40, 70, put(a), out, x_stride=72, out_stride=72, seed=seed, dropped=32768)
        hipmem.synchronize()
        outs.append(out.to_host().astype(np.float64))
    assert (y * outs[0]).sum() == (x * outs[1]).sum() != 0


# ---- together ----

@pytest.mark.parametrize("element", ["f32", "bf16"])
def test_a_step_captured_and_replayed(device, element):
    """Attention, dropout onto a residual, its backward pass and attention's, in one graph of a stream of its own: replayed
    with eager work between, each replay with the seed that stands in memory then."""
    case = Case(device, 2, 4, 2, 100, 700, element, "heads", (100, 60), (700, 300), random_keep(2, 700, 2), 6554)
    rows, width = 2 * 4 * 100, 64
    residual, mixed = (put(encode(normal((rows, width), 60 + i), element)) for i in (1, 2))
    back = put(encode(normal((rows, width), 63), element))
    rt = hipmem.runtime()
    for name in ("hipStreamCreate", "hipStreamBeginCapture", "hipStreamEndCapture", "hipGraphInstantiate", "hipGraphLaunch",
                 "hipStreamSynchronize", "hipStreamDestroy"):
        getattr(rt, name).restype = ctypes.c_int
    stream = ctypes.c_void_p()
    assert rt.hipStreamCreate(ctypes.byref(stream)) == 0
    drop = {"element": element, "seed": case.kept[3], "site": 9, "dropped": 6554}

    def step(on):
        case.forward(on)
        training.dropout(device, rows, width, case.out.array, mixed, residual=residual, stream=on, **drop)
        training.dropout(device, rows, width, back, case.dout.array, stream=on, **drop)
        case.backward(on)

    def results():
        hipmem.synchronize()
        return case.results() + [mixed.to_host(), case.dout.array.to_host()]

    # Rows past the lengths are not written by attention: they start as zeros for the dropout that reads them.
    case.out = Tensor((2, 4, 100, 64), element, "heads", np.zeros((2, 4, 100, 64)))
    step(None)
    eager = results()
    assert rt.hipStreamBeginCapture(stream, 0) == 0
    step(stream.value)
    graph, runnable = ctypes.c_void_p(), ctypes.c_void_p()
    assert rt.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert rt.hipGraphInstantiate(ctypes.byref(runnable), graph, None, None, ctypes.c_size_t(0)) == 0
    other = Case(device, 1, 2, 2, 30, 400, element)
    for number in (SEED, 12345, SEED):
        new = np.array([number], np.uint64)
        assert rt.hipMemcpy(case.kept[3].ptr, new.ctypes.data, 8, hipmem.H2D) == 0
        assert rt.hipGraphLaunch(runnable, stream) == 0
        assert rt.hipStreamSynchronize(stream) == 0
        got = results()
        other.check(other.run())
        same = [np.array_equal(x, y) for x, y in zip(got, eager)]
        assert all(same) if number == SEED else not any(same[i] for i in (0, 3, 4, 5, 6, 7)), number
        if number != SEED:
            step(None)  # eagerly, with that seed
            for x, y in zip(got, results()):
                np.testing.assert_array_equal(x, y)
    assert rt.hipStreamDestroy(stream) == 0


def test_refused_calls_leave_everything(device):
    case = Case(device, 1, 2, 2, 5, 2000)
    for space in (case.space[0], case.space[1]):
        assert space["workspace_bytes"] > 0
        space["workspace_bytes"] -= 16
    for call in (case.forward, case.backward):
        with pytest.raises(hip.HipError, match="the workspace must hold") as info:
            call()
        assert info.value.status == hip.INVALID_ARGUMENT
    hipmem.synchronize()
    for x in case.results():
        assert np.all(x == MARK)
