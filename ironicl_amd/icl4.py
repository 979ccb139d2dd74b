"""The 4-bit ICL cache on device buffers (irx_icl4_*, include/ironicl_hip.h).

Keys and values of 64-wide heads in 4 bits, attention over all of them, and
attention over the blocks of 64 rows that a cheap score picks for each query.

A buffer is an integer address, a ``hipmem.DeviceArray`` or anything with
``data_ptr()`` (a torch tensor on the device), or None where the call allows
it. Buffers are the caller's: they must be of the stated type and size, and
live until the work on ``stream`` (an address, or None for the null stream)
is done. ``shape`` is (estimators, heads, rows); strides are (estimator, head,
row) in elements, by default those of [estimators, heads, rows, 64]. Calls
enqueue their work and return; invalid ones raise ``hip.HipError``.
"""

from __future__ import annotations

import functools
import struct

from . import hip

ELEMENTS = {"f32": hip.ELEMENT_F32, "f16": hip.ELEMENT_F16}
BLOCK = 64  # rows of a block

# hip.Icl4Rows and hip.Icl4Queries as bytes: packing them costs a call a few
# microseconds less than building the structures field by field.
_ROWS = struct.Struct("@NNNiPPNNNNNNP")
_QUERIES = struct.Struct("@NNNNiPNNNPP")
_THREE = struct.Struct("@NNN")


def _address(buffer):
    if buffer is None or buffer.__class__ is int:
        return buffer
    try:
        return buffer.data_ptr()
    except AttributeError:
        return buffer.ptr


def _element(element: str) -> int:
    if element not in ELEMENTS:
        raise ValueError(f"element must be one of {sorted(ELEMENTS)}, not {element!r}")
    return ELEMENTS[element]


def _strides(strides, heads: int, rows: int):
    return (heads * rows * 64, rows * 64, 64) if strides is None else strides


def _refused() -> hip.HipError:
    return hip.HipError(hip.INVALID_ARGUMENT, "sizes and strides are whole numbers from 0 to 2^64 - 1")


def _size(n) -> int:
    # A size_t argument would take what lies outside modulo 2^64.
    try:
        n = n.__index__()
    except AttributeError:
        raise _refused() from None
    if not 0 <= n < 1 << 64:
        raise _refused()
    return n


def _rows(shape, k, v, element, k_strides, v_strides, lengths) -> bytes:
    estimators, heads, rows = shape
    try:
        return _ROWS.pack(estimators, heads, rows, _element(element), _address(k) or 0, _address(v) or 0,
                          *_strides(k_strides, heads, rows), *_strides(v_strides, heads, rows), _address(lengths) or 0)
    except struct.error:
        raise _refused() from None


def _queries(shape, q, query_rows, element, q_strides, lengths, keep) -> bytes:
    estimators, heads, rows = shape
    try:
        return _QUERIES.pack(estimators, heads, rows, query_rows, _element(element), _address(q) or 0,
                             *_strides(q_strides, heads, query_rows), _address(lengths) or 0, _address(keep) or 0)
    except struct.error:
        raise _refused() from None


@functools.lru_cache(maxsize=None)
def _call(name: str):
    return getattr(hip.lib(), name)


def _shape(shape) -> bytes:  # hip.Icl4Shape, or hip.Strides
    try:
        return _THREE.pack(*shape)
    except struct.error:
        raise _refused() from None


def cache_bytes(shape) -> int:
    """Bytes of a cache of `shape` (0: out of range)."""
    try:
        return _call("irx_icl4_bytes")(_shape(shape))
    except hip.HipError:
        return 0


def workspace_bytes(device: hip.Device, shape, query_rows: int, n_blocks: int = 0) -> int:
    """Bytes of workspace for `select` and `attention` of exactly `query_rows` queries
    (fewer can need more: they are split further) over `n_blocks` blocks each, or all.
    0 where none is needed, and for arguments out of range, which the calls refuse."""
    try:
        return _call("irx_icl4_workspace_bytes")(device.handle, _shape(shape), _size(query_rows), _size(n_blocks))
    except hip.HipError:
        return 0


def encode(device: hip.Device, shape, k, v, cache, *, element: str = "f32", k_strides=None, v_strides=None,
           lengths=None, nonfinite=None, stream=None) -> None:
    """Writes `cache` (cache_bytes) from keys and values [estimators, heads, rows, 64];
    numbers that are not finite are held as 0 and added to the uint32 `nonfinite`."""
    rows = _rows(shape, k, v, element, k_strides, v_strides, lengths)
    hip.check(_call("irx_icl4_encode")(device.handle, rows, _address(cache), _address(nonfinite), _address(stream)))


def decode(device: hip.Device, shape, cache, k=None, v=None, *, element: str = "f32", k_strides=None,
           v_strides=None, lengths=None, bounds=None, stream=None) -> None:
    """Reads what `cache` holds into k and v, and its bounds into FP32 [estimators *
    heads, blocks, 2, 64]. Rows past an estimator's length are left as they were."""
    rows = _rows(shape, k, v, element, k_strides, v_strides, lengths)
    hip.check(_call("irx_icl4_decode")(device.handle, _address(cache), rows, _address(bounds), _address(stream)))


def select(device: hip.Device, shape, cache, q, query_rows: int, n_blocks: int, blocks, *, element: str = "f32",
           q_strides=None, lengths=None, keep=None, workspace=None, workspace_bytes: int = 0, stream=None) -> None:
    """The `n_blocks` best blocks of each query into int32 `blocks` [estimators,
    heads, query_rows, n_blocks], ascending, -1 where there are fewer."""
    queries = _queries(shape, q, query_rows, element, q_strides, lengths, keep)
    hip.check(_call("irx_icl4_select")(device.handle, queries, _address(cache), _size(n_blocks), _address(blocks),
                                       _address(workspace), _size(workspace_bytes), _address(stream)))


def attention(device: hip.Device, shape, cache, q, query_rows: int, out, *, element: str = "f32", scale: float = 0.125,
              q_strides=None, out_strides=None, lengths=None, keep=None, blocks=None, n_blocks: int = 0, lse=None,
              workspace=None, workspace_bytes: int = 0, stream=None) -> None:
    """softmax(scale q k^T) v over the attended rows (those of `blocks`, when
    given) into `out`, and the log-sum-exp into FP32 `lse` [estimators, heads,
    query_rows]; 0 and -inf where a query attends to nothing."""
    queries = _queries(shape, q, query_rows, element, q_strides, lengths, keep)
    strides = _shape(_strides(out_strides, shape[1], query_rows))
    hip.check(_call("irx_icl4_attention")(device.handle, queries, _address(cache), scale, _address(blocks),
                                          _size(n_blocks), _address(out), strides, _address(lse), _address(workspace),
                                          _size(workspace_bytes), _address(stream)))
