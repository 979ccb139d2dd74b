"""The training calls without a GPU: what they refuse before they touch the device, and the oracle itself."""

import ctypes

import numpy as np
import pytest

import training_np
from ironicl_amd import hip, training

SHAPE = (1, 8, 2, 33, 100)
Q = 1 << 20  # an aligned address that is never read: every call here is refused


class NoDevice:
    handle = None


def refused(text, call, *args, **kw):
    with pytest.raises(hip.HipError, match=text) as info:
        call(NoDevice(), *args, **kw)
    assert info.value.status == hip.INVALID_ARGUMENT


def test_structures_are_the_headers():
    for packed, declared in ((training._SHAPE, hip.TrainShape), (training._INPUTS, hip.TrainInputs),
                             (training._GRADIENTS, hip.TrainGradients), (training._ROWS, hip.TrainRows)):
        assert packed.size == ctypes.sizeof(declared)


def test_attention_is_checked():
    call = training.attention
    refused("needs its inputs and its output", call, SHAPE, Q, Q, Q, None)
    for i in range(3):
        refused("needs queries, keys and values", call, SHAPE, *[None if j == i else Q for j in range(3)], Q)
    for shape in ((0, 8, 2, 33, 100), (1, 0, 2, 33, 100), (1, 8, 0, 33, 100), (1, 8, 2, 0, 100), (1, 8, 2, 33, 0),
                  (65536, 1, 1, 1, 1), (1024, 64, 1, 1, 1), (1, 8, 3, 33, 100), (1, 8, 16, 33, 100),
                  (1, 1, 1, (1 << 24) + 1, 1), (1, 1, 1, 1, (1 << 24) + 1), (1 << 40, 1 << 40, 1, 1, 1)):
        refused("shape is out of range", call, shape, Q, Q, Q, Q)
    for scale in (0.0, -1.0, 2.0 ** -65, 2.0 ** 65, 1e39, float("inf"), float("nan")):
        refused("the scale is 2\\^-64 to 2\\^64", call, SHAPE, Q, Q, Q, Q, scale=scale)
    refused("queries must be aligned to 16", call, SHAPE, Q + 8, Q, Q, Q)
    refused("keys must be aligned to 16", call, SHAPE, Q, Q + 4, Q, Q)
    refused("values must be aligned to 16", call, SHAPE, Q, Q, Q + 2, Q)
    refused("the output must be aligned to 16", call, SHAPE, Q, Q, Q, Q + 1)
    refused("stats must be aligned to 8", call, SHAPE, Q, Q, Q, Q, stats=Q + 4)
    refused("lse must be aligned to 4", call, SHAPE, Q, Q, Q, Q, lse=Q + 2)
    refused("keep must be aligned to 8", call, SHAPE, Q, Q, Q, Q, keep=Q + 4)
    refused("query lengths must be aligned to 4", call, SHAPE, Q, Q, Q, Q, query_lengths=Q + 2)
    refused("lengths must be aligned to 4", call, SHAPE, Q, Q, Q, Q, lengths=Q + 1)
    refused("multiples of 16 bytes", call, SHAPE, Q, Q, Q, Q, k_strides=(0, 6400, 66))
    refused("multiples of 16 bytes", call, SHAPE, Q, Q, Q, Q, element="bf16", q_strides=(0, 6400, 68))
    refused("within range", call, SHAPE, Q, Q, Q, Q, v_strides=(0, 1 << 60, 64))
    refused("must not overlap", call, SHAPE, Q, Q, Q, Q, out_strides=(0, 64, 64))
    refused("dropout needs a seed", call, SHAPE, Q, Q, Q, Q, dropped=1)
    refused("0 to 65,535", call, SHAPE, Q, Q, Q, Q, seed=Q, dropped=65536)
    refused("the seed must be aligned to 8", call, SHAPE, Q, Q, Q, Q, seed=Q + 4, dropped=1)
    refused("needs a device", call, SHAPE, Q, Q, Q, Q, k_strides=(0, 0, 0), seed=Q, dropped=65535, scale=2.0 ** 64)
    with pytest.raises(ValueError, match="element must be one of"):
        call(NoDevice(), SHAPE, Q, Q, Q, Q, element="f64")


def test_the_backward_pass_is_checked():
    call = training.attention_backward
    six = [Q] * 6
    for i in range(3, 6):
        refused("needs its inputs, the output, its statistics and its gradient", call, SHAPE,
                *[None if j == i else Q for j in range(6)], dq=Q)
    for sides in ({}, {"dk": Q}, {"dv": Q}, {"dq": Q, "dv": Q}, {"dq": Q, "dk": Q}):
        refused("gradients are of the queries, of keys and values, or of both", call, SHAPE, *six, **sides)
    every = {"dq": Q, "dk": Q, "dv": Q}
    refused("shape is out of range", call, (1, 8, 3, 33, 100), *six, **every)
    refused("must not overlap", call, SHAPE, *six, **every, dq_strides=(0, 64, 64))
    refused("must not overlap", call, SHAPE, *six, **every, dk_strides=(0, 0, 64))
    refused("must not overlap", call, SHAPE, *six, **every, dv_strides=(0, 6400, 0))
    for name, text in (("dq", "the queries' gradient"), ("dk", "the keys' gradient"), ("dv", "the values' gradient")):
        refused(text + " must be aligned to 16", call, SHAPE, *six, **dict(every, **{name: Q + 8}))
    refused("the output's gradient must be aligned to 16", call, SHAPE, Q, Q, Q, Q, Q, Q + 8, **every)
    refused("stats must be aligned to 8", call, SHAPE, Q, Q, Q, Q, Q + 4, Q, **every)
    refused("dropout needs a seed", call, SHAPE, *six, **every, dropped=7)
    refused("needs a device", call, SHAPE, *six, **every)
    refused("needs a device", call, SHAPE, *six, dq=Q)
    refused("needs a device", call, SHAPE, *six, dk=Q, dv=Q, dk_strides=(0, 64, 128), dout_strides=(0, 0, 0))


def test_dropout_is_checked():
    call = training.dropout
    refused("needs its input and its output", call, 4, 8, None, Q)
    refused("needs its input and its output", call, 4, 8, Q, None)
    for rows, width in ((0, 8), (8, 0), (1, 1 << 31), (1 << 31, 1), (1 << 28, 64)):
        refused("rows and columns are out of range", call, rows, width, Q, Q, x_stride=64, out_stride=64)
    refused("a tensor must be aligned to 16", call, 4, 8, Q + 4, Q)
    refused("a tensor must be aligned to 16", call, 4, 8, Q, Q, residual=Q + 8)
    refused("the width at least", call, 4, 12, Q, Q, x_stride=8)
    refused("multiples of 16 bytes", call, 4, 13, Q, Q)
    refused("multiples of 16 bytes", call, 4, 12, Q, Q, element="f16")
    refused("within range", call, 4, 8, Q, Q, out_stride=1 << 40)
    refused("dropout needs a seed", call, 4, 8, Q, Q, dropped=1)
    refused("an input that is the output", call, 4, 8, Q, Q, x_stride=16)
    refused("an input that is the output", call, 4, 8, Q, Q + 64, residual=Q + 64, out_stride=16)
    refused("needs a device", call, 4, 8, Q, Q + 64, residual=Q, x_stride=16)
    refused("needs a device", call, 1, 13, Q, Q)
    refused("needs a device", call, 4, 12, Q, Q, residual=Q, seed=Q, dropped=65535)
    with pytest.raises(ValueError, match="element must be one of"):
        call(NoDevice(), 4, 8, Q, Q, element="f8")


def test_numbers_that_are_no_sizes_are_refused():
    device = NoDevice()
    calls = [
        lambda: training.attention(device, (1, 8, 2, -33, 100), Q, Q, Q, Q),
        lambda: training.attention(device, (1, 8, 2, 33, 1 << 64), Q, Q, Q, Q),
        lambda: training.attention(device, SHAPE, Q, Q, Q, Q, k_strides=(0, -64, 64)),
        lambda: training.attention(device, SHAPE, Q, Q, Q, Q, out_strides=(0, 64, -512)),
        lambda: training.attention(device, SHAPE, Q, Q, Q, Q, dropped=-1, seed=Q),
        lambda: training.attention(device, SHAPE, Q, Q, Q, Q, dropped=1 << 32, seed=Q),
        lambda: training.attention(device, SHAPE, Q, Q, Q, Q, site=-1),
        lambda: training.attention(device, SHAPE, Q, Q, Q, Q, workspace=Q, workspace_bytes=-1),
        lambda: training.attention_backward(device, SHAPE, *[Q] * 6, dq=Q, workspace=Q, workspace_bytes=1 << 64),
        lambda: training.attention_backward(device, SHAPE, *[Q] * 6, dq=Q, dq_strides=(0, 64, 1.5)),
        lambda: training.dropout(device, -1, 8, Q, Q),
        lambda: training.dropout(device, 4, 8, Q, Q, out_stride=-8),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(hip.HipError, match="sizes and strides are whole numbers") as info:
            call()
        assert info.value.status == hip.INVALID_ARGUMENT, i
    for shape in ((1, 8, 2, -1, 100), (1, 8, 2, 1 << 64, 100), (1, 8, 2, 1.5, 100), SHAPE):
        assert training.workspace_bytes(device, shape) == 0


def test_null_and_unknown_arguments_are_errors():
    lib = hip.lib()
    assert lib.irx_train_attention(None, None, Q, None, None, None, None, 0, None) == hip.INVALID_ARGUMENT
    assert lib.irx_train_attention_backward(None, None, None, None, 0, None) == hip.INVALID_ARGUMENT
    assert lib.irx_train_dropout(None, None, None) == hip.INVALID_ARGUMENT
    assert lib.irx_train_workspace_bytes(None, None, 0, 0) == 0
    rows = hip.TrainRows(1, 8, 3, Q, None, Q, 8, 8, 8, hip.TrainDrop(None, 0, 0))
    assert lib.irx_train_dropout(None, ctypes.byref(rows), None) == hip.INVALID_ARGUMENT
    assert b"FP32, FP16 or BF16" in lib.irx_last_error()


def test_the_4_bit_cache_takes_no_bf16():
    queries = hip.Icl4Queries(hip.Icl4Shape(1, 8, 100), 1, hip.ELEMENT_BF16, Q, hip.Strides(0, 64, 64), None, None)
    out = hip.Strides(0, 64, 64)
    assert hip.lib().irx_icl4_attention(None, ctypes.byref(queries), Q, 1.0, None, 0, Q, ctypes.byref(out), None, None,
                                        0, None) == hip.INVALID_ARGUMENT
    assert b"FP32 or FP16" in hip.lib().irx_last_error()


# ---- the oracle ----

def test_philox_known_answers():
    """The paper's authors publish these with their library for ten rounds (counter, key: zeros; all ones)."""
    words = [int(x) for x in training_np.philox((0, 0, 0, 0), (0, 0), rounds=10)]
    assert words == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = 0xFFFFFFFF
    words = [int(x) for x in training_np.philox((ones,) * 4, (ones, ones), rounds=10)]
    assert words == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


def test_dropout_drops_as_many_as_it_says_and_no_pattern():
    for dropped in (655, 6554, 32768):
        p = dropped / 65536
        for kept in (training_np.kept_weights(7, 0, dropped, 3, 700, 900), training_np.kept_numbers(7, 0, dropped, 700, 900)):
            drop = 1.0 - kept
            n = drop.size
            assert abs(drop.mean() - p) < 5 * np.sqrt(p * (1 - p) / n)
            # Rows, columns, and neighbours of either side are as independent numbers are (5 standard deviations).
            for axis in (0, 1):
                spread = drop.mean(axis).std() / np.sqrt(p * (1 - p) / drop.shape[axis])
                assert abs(spread - 1) < 5 / np.sqrt(2 * drop.shape[1 - axis])
                for step in (1, 2, 4, 8, 16, 32):
                    a, b = np.delete(drop, np.s_[-step:], axis), np.delete(drop, np.s_[:step], axis)
                    assert abs(((a - p) * (b - p)).mean()) < 5 * p * (1 - p) / np.sqrt(a.size)
    a, b, c = (training_np.kept_weights(seed, site, 32768, pair, 200, 200) for seed, site, pair in ((7, 0, 0), (7, 1, 0), (8, 0, 1)))
    for x, y in ((a, b), (a, c), (b, c)):
        assert abs((x == y).mean() - 0.5) < 0.0125  # 5 standard deviations


def test_the_oracles_gradients_against_differences():
    rng = np.random.default_rng(0)
    q, k, v, dout = rng.normal(size=(2, 4, 6, 64)), rng.normal(size=(2, 2, 30, 64)), rng.normal(size=(2, 2, 30, 64)), rng.normal(size=(2, 4, 6, 64))
    args = dict(q_lengths=np.array([6, 4]), lengths=np.array([30, 11]), keep=rng.random((2, 30)) < 0.7, seed=9, site=2, dropped=20000)
    want = training_np.Attention(q, k, v, dout=dout, **args)
    for i, grad in enumerate((want.dq, want.dk, want.dv)):
        step = rng.normal(size=grad.shape) * 1e-5
        loss = [(training_np.Attention(*[x + s * step if j == i else x for j, x in enumerate((q, k, v))], **args).out * dout).sum() for s in (1, -1)]
        assert abs((loss[0] - loss[1]) / 2 - (grad * step).sum()) < 1e-9 * np.abs(grad * step).sum() + 1e-13
