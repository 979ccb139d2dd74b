"""The training calls at the ends of their ranges, against float64 (training_np.py) within the bounds that
test_gpu_training.py works out: numbers far below 1, and far above it beside others; only what a test adds to them stands there."""

import numpy as np
import pytest

import training_np
from ironicl_amd import hip, hipmem, training
from test_gpu_training import HALF, PARTS, SEED, Case, decode, encode, floor, normal, put, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def device():
    return hip.Device(0)


def bounds(case, want, ds, key_ds=None):
    """Bounds of out, dq, dk and dv where every score is off by ds (in the keys' sums by key_ds)."""
    el, (_, h, g, m, n) = case.element, case.shape
    m *= h // g
    key_ds = ds if key_ds is None else key_ds
    forward = 2 * ds + PARTS[el] + n * 2.0 ** -26 + 2.0 ** -20
    gradient = 2 * PARTS[el] + 2.0 ** -17 + forward + HALF[el] + 2.0 ** -19
    return (want.out_abs * forward + floor(want.out_term, n, el),
            want.dq_abs * (gradient + 2 * ds + n * 2.0 ** -26) + floor(want.dq_term, n, el),
            want.dk_abs * (gradient + 2 * key_ds + m * 2.0 ** -26) + floor(want.dk_term, m, el),
            want.dv_abs * (2 * key_ds + PARTS[el] + m * 2.0 ** -26 + 2.0 ** -20) + floor(want.dv_term, m, el))


def compare(case, got, want, ds, key_ds=None):
    exact = (want.out, want.dq, want.dk, want.dv)
    for name, have, x, bound in zip(("out", "dq", "dk", "dv"), [got[0]] + got[3:], exact, bounds(case, want, ds, key_ds)):
        within(have, x, bound, np.ones(have.shape, bool), case.element, name)


@pytest.mark.parametrize("dropped", [0, 3000])
@pytest.mark.parametrize("values,gradients", [(0, -100), (0, -108), (-50, -55), (-55, -50), (40, -108)])
def test_fp32_gradients_of_small_products(device, values, gradients, dropped):
    """dout and v by powers of two: dq and dk by their product, dv by dout's, though dP is far below 1. Each of 130 terms may
    miss 2^-126 times an operand up to 8, and a sum that misses one may round the other way once in each of its additions,
    fewer than 64, by 2^-24 of a sum of magnitudes."""
    dout, v = normal((1, 2, 70, 64), 3), normal((1, 2, 130, 64), 2)
    a = Case(device, 1, 2, 2, 70, 130, dropped=dropped, seed=4, dout=dout, v=v)
    b = Case(device, 1, 2, 2, 70, 130, dropped=dropped, seed=4, dout=a.dout.values * 2.0 ** gradients, v=a.v.values * 2.0 ** values)
    want, first, second = a.oracle(), a.run(), b.run()
    np.testing.assert_array_equal(first[0] * 2.0 ** values, second[0])
    for name, x, y, by, size in zip(("dq", "dk", "dv"), first[3:], second[3:], (values + gradients,) * 2 + (gradients,),
                                    (want.dq_abs, want.dk_abs, want.dv_abs)):
        off = np.abs(x * 2.0 ** by - y) - (size * 2.0 ** (by - 18) + 130 * 8 * 2.0 ** -126)
        assert off.max() <= 0, f"{name} past the bound by {off.max():.3e}"


def test_fp32_gradients_of_large_rows(device):
    """Rows of v whose largest number meets a zero of dout: dP is within FP32's range though its row times dout's is not."""
    rng = np.random.default_rng(5)
    v, dout = np.zeros((1, 2, 200, 64)), np.zeros((1, 2, 40, 64))
    v[..., 0] = 2.0 ** 120 * rng.choice([-1.0, 1.0], (1, 2, 200))
    v[..., 1] = 2.0 ** 85 * rng.choice([-1.0, 1.0], (1, 2, 200))
    dout[..., 1] = 2.0 ** 40 * rng.choice([-1.0, 1.0], (1, 2, 40))
    case = Case(device, 1, 2, 2, 40, 200, v=v, dout=dout)
    got, want = case.run(), case.oracle()
    compare(case, got, want, 2.0 ** -17 * want.magnitude.max())


@pytest.mark.parametrize("at", [0, 20, 299])
@pytest.mark.parametrize("queries", [9, 40, 130])
@pytest.mark.parametrize("element", ["f32", "bf16"])
@pytest.mark.parametrize("size,score", [(60, -1000), (80, -1000), (120, -1000), (80, -62), (120, -40), (126, -12)])
def test_small_values_beside_a_large_one(device, size, score, element, queries, at):
    """One value of 2^size whose score lies far below the others': of no weight, of as much as the others have together, or of
    so much more that they hardly show, but in the sums of weights. It is in the first tile, beside them, or in the last."""
    e, h, n = 1, 2, 300
    q, k, v = normal((e, h, queries, 64), 1, 1.3), normal((e, h, n, 64), 2, 1.1), normal((e, h, n, 64), 3)
    q[..., 0], k[..., 0] = 8.0, 0.0
    k[:, :, at] = 0.0
    k[:, :, at, 0], v[:, :, at, 5] = score, 2.0 ** size
    dout = normal(q.shape, 4, 2.0 ** -6)
    case = Case(device, e, h, h, queries, n, element, q=q, k=k, v=v, dout=dout)
    got, want = case.run(), case.oracle()
    # Its score is a whole number; at no weight, the others' alone count.
    keep = np.arange(n) != at
    others = training_np.Attention(case.q.values, case.k.values, case.v.values, keep=keep[None])
    ds = 2.0 ** -17 * (others.magnitude.max() + (-score if score > -1000 else 0))
    compare(case, got, want, ds)
    off = np.abs(got[1] - want.lse) - (2 * ds + n * 2.0 ** -26 + 2.0 ** -21 * np.abs(want.lse) + 1e-6)
    assert off.max() <= 0


@pytest.mark.parametrize("dropped", [0, 9000])
@pytest.mark.parametrize("element", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("queries", [1, 3, 40, 200])
@pytest.mark.parametrize("size", [2.0 ** 5, 2.0 ** 8, 2.0 ** 13, 2.0 ** 20])
def test_scores_that_are_whole_at_any_size(device, size, queries, element, dropped):
    """Products of queries and keys are whole numbers below 2^24, and their sums in any order: scores differ by a few either
    way at sizes up to 2^20. log2(e) scale is off by 2^-24 of itself, and so are differences of scores; a score's distance
    from its reference (24 at most, where its weight counts) is rounded once, to 2^-24 of it: 2^-19 in all, with a step to
    spare. In the sums of 16-bit types' keys, references below 2^7 stand as one number with their sums' logarithms: 16
    roundings of it at most, 2^-13."""
    e, h, n = 1, 2, 300
    rng = np.random.default_rng(int(size))
    q, k = (rng.integers(-2, 3, (e, h, rows, 64)).astype(float) for rows in (queries, n))
    q[..., 0] = 2.0 ** 12 * rng.choice([-1.0, 1.0], (e, h, queries))
    k[..., 0] = size * 2.0 ** -9 * rng.choice([-1.0, 1.0], (e, h, n))
    case = Case(device, e, h, h, queries, n, element, q=q, k=k, scale=2.0 ** -3, dropped=dropped)
    got, want = case.run(), case.oracle()
    assert want.lse.min() > size - 20
    few = element != "f32" and size < 2.0 ** 6
    compare(case, got, want, 2.0 ** -19, 2.0 ** -13 if few else None)
    assert np.all(np.abs(got[1] - want.lse) <= 2.0 ** -22 * np.abs(want.lse) + n * 2.0 ** -26 + 2.0 ** -18)


@pytest.mark.parametrize("element", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dropped", [0, 1, 6554, 40001, 65535])
def test_dropout_is_one_multiplication_and_addition(device, dropped, element):
    """x w + residual, rounded once to FP32 and then to the type. x and residual are multiples of 2^-3 and 2^-10 below 2^4,
    so that float64 holds the products with w's 24 bits, and the sums, whole."""
    rng = np.random.default_rng(dropped)
    rows, width = 300, 136
    x = rng.integers(-127, 128, (rows, width)) * 2.0 ** -3
    residual = rng.integers(-127, 128, (rows, width)) * 2.0 ** -10
    seed, out = put(np.array([SEED], np.uint64)), put(encode(np.zeros((rows, width)), element))
    w = float(np.float32(65536.0) / np.float32(65536 - dropped))
    term = x * w * training_np.kept_numbers(SEED, 7, dropped, rows, width)
    for second in (None, residual):
        training.dropout(device, rows, width, put(encode(x, element)), out, element=element,
                         residual=None if second is None else put(encode(second, element)), seed=seed, site=7, dropped=dropped)
        hipmem.synchronize()
        want = encode((term + (0.0 if second is None else second)).astype(np.float32), element)
        np.testing.assert_array_equal(decode(out.to_host(), element), decode(want, element))


@pytest.mark.parametrize("queries", [1, 8, 40, 200])
def test_fp32_products_keep_their_lower_halves(device, queries):
    """Numbers whose bits past the eleventh all point one way: a product of a lower with an upper half that went missing
    would show in every score, weight and gradient at once (64 terms of 2^-12, one sign)."""
    def numbers(shape, seed):
        rng = np.random.default_rng(seed)
        # 1 to 2 in steps of 2^-10, and half a step more: the half step is the lower half.
        return 1.0 + (rng.integers(0, 1024, shape) + 0.5) * 2.0 ** -10 - 2.0 ** -22

    e, h, n = 1, 2, 300
    signs = [np.random.default_rng(i).choice([-1.0, 1.0], (e, h, rows, 1)) for i, rows in ((9, n), (10, queries))]
    case = Case(device, e, h, h, queries, n, q=numbers((e, h, queries, 64), 1), k=numbers((e, h, n, 64), 2) * signs[0],
                v=numbers((e, h, n, 64), 3), dout=numbers((e, h, queries, 64), 4) * signs[1], scale=2.0 ** -7)
    got, want = case.run(), case.oracle()
    compare(case, got, want, 2.0 ** -17 * want.magnitude.max())
    # A score is |scale q k| <= 2: two lower halves' product left out and two rounded, 2^-22 each, and sums of 2^-18 of it.
    assert np.all(np.abs(got[1] - want.lse) <= 2.0 ** -16 + n * 2.0 ** -26)
