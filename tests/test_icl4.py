"""The 4-bit ICL cache without a GPU: its sizes, and the calls it refuses
before it touches the device."""

import ctypes

import numpy as np
import pytest

import icl4_np
from ironicl_amd import hip, icl4

SHAPE = (1, 8, 100)
Q = 1 << 20  # an aligned address that is never read: every call here is refused


def refused(text, call, *args, **kw):
    with pytest.raises(hip.HipError, match=text) as info:
        call(None_device(), *args, **kw)
    assert info.value.status == hip.INVALID_ARGUMENT


class None_device:
    handle = None


def test_cache_bytes():
    assert icl4.cache_bytes((1, 8, 64)) == 8 * 4480 + 8 * 256
    assert icl4.cache_bytes((2, 8, 65)) == 16 * 2 * 4480 + 16 * 256
    assert icl4.cache_bytes((1, 1, 1)) == 4480 + 256
    for shape in ((0, 8, 64), (1, 0, 64), (1, 8, 0), (65536, 1, 1), (1, 1, (1 << 27) + 1), (65535, 1, 1 << 27)):
        assert icl4.cache_bytes(shape) == 0
    assert hip.lib().irx_icl4_bytes(None) == 0
    assert hip.lib().irx_icl4_workspace_bytes(None, ctypes.byref(hip.Icl4Shape(*SHAPE)), 1, 0) == 0


def test_rows_are_checked():
    refused("written from keys and values", icl4.encode, SHAPE, None, Q, Q)
    refused("written from keys and values", icl4.encode, SHAPE, Q, Q, None)
    refused("shape is out of range", icl4.encode, (0, 8, 100), Q, Q, Q)
    refused("keys must be aligned to 16", icl4.encode, SHAPE, Q + 8, Q, Q)
    refused("values must be aligned to 16", icl4.encode, SHAPE, Q, Q + 4, Q)
    refused("the cache must be aligned", icl4.encode, SHAPE, Q, Q, Q + 8)
    refused("lengths must be aligned", icl4.encode, SHAPE, Q, Q, Q, lengths=Q + 2)
    refused("the counter must be aligned", icl4.encode, SHAPE, Q, Q, Q, nonfinite=Q + 1)
    refused("multiples of 16 bytes", icl4.encode, SHAPE, Q, Q, Q, k_strides=(0, 6400, 66))
    refused("multiples of 16 bytes", icl4.encode, SHAPE, Q, Q, Q, element="f16", v_strides=(0, 6400, 68))
    refused("within range", icl4.encode, SHAPE, Q, Q, Q, k_strides=(0, 1 << 60, 64))
    refused("needs a device", icl4.encode, SHAPE, Q, Q, Q)
    refused("needs a device", icl4.encode, SHAPE, Q, Q, Q, k_strides=(0, 0, 0), v_strides=(7, 0, 64))
    refused("nothing to read", icl4.decode, SHAPE, Q)
    refused("must not overlap", icl4.decode, SHAPE, Q, k=Q, k_strides=(0, 64, 64))
    refused("must not overlap", icl4.decode, SHAPE, Q, v=Q, v_strides=(0, 0, 64))
    refused("must not overlap", icl4.decode, (2, 8, 100), Q, v=Q, v_strides=(512 * 99, 64, 512))
    refused("needs a device", icl4.decode, (2, 8, 100), Q, v=Q, v_strides=(512 * 100, 64, 512))
    refused("needs a device", icl4.decode, SHAPE, Q, bounds=Q)
    with pytest.raises(ValueError, match="element must be one of"):
        icl4.encode(None_device(), SHAPE, Q, Q, Q, element="bf16")


def test_queries_are_checked():
    refused("needs queries, a cache and its output", icl4.select, SHAPE, None, Q, 1, 1, Q)
    refused("1 to 4096 blocks", icl4.select, SHAPE, Q, Q, 1, 0, Q)
    refused("1 to 4096 blocks", icl4.select, SHAPE, Q, Q, 1, 4097, Q)
    refused("1 to 2\\^24 queries", icl4.select, SHAPE, Q, Q, 0, 1, Q)
    refused("1 to 2\\^24 queries", icl4.select, SHAPE, Q, None, 1, 1, Q)
    refused("too many queries", icl4.select, (1024, 8, 100), Q, Q, 1 << 24, 1, Q)
    refused("keep must be aligned to 8", icl4.select, SHAPE, Q, Q, 1, 1, Q, keep=Q + 4)
    refused("needs a device", icl4.select, SHAPE, Q, Q, 1, 1, Q)
    refused("needs queries, a cache and its output", icl4.attention, SHAPE, Q, Q, 1, None)
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        refused("positive and finite", icl4.attention, SHAPE, Q, Q, 1, Q, scale=scale)
    refused("name 1 to 4096 blocks", icl4.attention, SHAPE, Q, Q, 1, Q, blocks=Q)
    refused("name 1 to 4096 blocks", icl4.attention, SHAPE, Q, Q, 1, Q, n_blocks=3)
    refused("queries must be aligned", icl4.attention, SHAPE, Q, Q + 8, 1, Q)
    refused("the output must be aligned", icl4.attention, SHAPE, Q, Q, 1, Q + 8)
    refused("multiples of 16 bytes", icl4.attention, SHAPE, Q, Q, 2, Q, out_strides=(0, 128, 66))
    refused("must not overlap", icl4.attention, SHAPE, Q, Q, 2, Q, out_strides=(0, 64, 64))
    refused("needs a device", icl4.attention, SHAPE, Q, Q, 2, Q, out_strides=(0, 64, 512))


def test_scales_past_the_largest_are_refused():
    for scale in (float.fromhex("0x1.000002p127"), 2.4e38, 3.4e38):
        refused("positive and finite, at most 2\\^127", icl4.attention, SHAPE, Q, Q, 1, Q, scale=scale)
    refused("needs a device", icl4.attention, SHAPE, Q, Q, 1, Q, scale=2.0 ** 127)


def test_numbers_that_are_no_sizes_are_refused():
    """Not passed on as the sizes that they would wrap to."""
    device = None_device()
    calls = [
        lambda: icl4.encode(device, (1, 8, -100), Q, Q, Q),
        lambda: icl4.encode(device, (1, 8, 1 << 64), Q, Q, Q),
        lambda: icl4.encode(device, SHAPE, Q, Q, Q, k_strides=(0, -64, 64)),
        lambda: icl4.decode(device, (-1, 8, 100), Q, k=Q),
        lambda: icl4.select(device, SHAPE, Q, Q, -1, 1, Q),
        lambda: icl4.select(device, SHAPE, Q, Q, 1, -1, Q),
        lambda: icl4.select(device, SHAPE, Q, Q, 1, (1 << 64) + 1, Q),
        lambda: icl4.select(device, SHAPE, Q, Q, 1, 1, Q, workspace=Q, workspace_bytes=-1),
        lambda: icl4.attention(device, SHAPE, Q, Q, 1.5, Q),
        lambda: icl4.attention(device, SHAPE, Q, Q, 2, Q, out_strides=(0, 64, -512)),
        lambda: icl4.attention(device, SHAPE, Q, Q, 1, Q, blocks=Q, n_blocks=-1),
        lambda: icl4.attention(device, SHAPE, Q, Q, 1, Q, workspace=Q, workspace_bytes=-1),
        lambda: icl4.attention(device, SHAPE, Q, Q, 1, Q, workspace=Q, workspace_bytes=1 << 64),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(hip.HipError, match="sizes and strides are whole numbers") as info:
            call()
        assert info.value.status == hip.INVALID_ARGUMENT, i
    for shape in ((1, 8, -64), (1, 8, 1 << 64), (1.5, 8, 64)):
        assert icl4.cache_bytes(shape) == 0
        assert icl4.workspace_bytes(device, shape, 1) == 0
    for rows, blocks in ((-1, 0), (1, -1), (1 << 64, 0), ((1 << 64) + 1, 0), (1, 1 << 64)):
        assert icl4.workspace_bytes(device, SHAPE, rows, blocks) == 0


def test_unknown_elements_are_refused():
    queries = hip.Icl4Queries(hip.Icl4Shape(*SHAPE), 1, 7, Q, hip.Strides(0, 64, 64), None, None)
    out = hip.Strides(0, 64, 64)
    assert hip.lib().irx_icl4_attention(None, ctypes.byref(queries), Q, 1.0, None, 0, Q, ctypes.byref(out), None, None,
                                        0, None) == hip.INVALID_ARGUMENT
    assert b"FP32 or FP16" in hip.lib().irx_last_error()


def test_codes_round_to_the_nearest_level_and_ties_to_the_even_code():
    """The oracle itself, on values worked out by hand: exponent 0 (a 6 in each group)."""
    x = np.zeros((1, 64, 64))
    x[0, 0, :10] = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0.26, -0.74, 6.0)
    c, e = icl4_np.codes(x, 2)
    assert list(c[0, 0, :10]) == [0, 2, 2, 4, 4, 6, 6, 1, 8 + 1, 7] and e[0, 0, 0] == 0
    assert icl4_np.unit(np.array([6.0, 6.01, 0.0, 1e9, 3e-5]), 6.0, -13, 13).tolist() == [0, 1, -13, 13, -13]
