"""Attention for training, its backward pass and dropout on device buffers
(irx_train_*, include/ironicl_hip.h).

A buffer is an integer address, a ``hipmem.DeviceArray`` or anything with
``data_ptr()`` (a torch tensor on the device), or None where the call allows
it. Buffers are the caller's: they must be of the stated type and size, and
live until the work on ``stream`` (an address, or None for the null stream)
is done. ``shape`` is (estimators, heads, kv_heads, query_rows, rows); strides
are (estimator, head, row) in elements, by default those of [estimators,
heads, rows, 64]. ``element`` is that of every tensor but FP32 ``stats`` and
``lse``. Dropout: ``dropped`` of 65,536 numbers become 0, which ones follows
from the uint64 at ``seed`` and from ``site``. Calls enqueue their work and
return; invalid ones raise ``hip.HipError``.
"""

from __future__ import annotations

import functools
import struct

from . import hip

ELEMENTS = {"f32": hip.ELEMENT_F32, "f16": hip.ELEMENT_F16, "bf16": hip.ELEMENT_BF16}

# hip.TrainInputs, hip.TrainGradients and hip.TrainRows as bytes: packing them
# costs a call less than building the structures field by field.
_SHAPE = struct.Struct("@NNNNN")
_INPUTS = struct.Struct("@NNNNNifPPPNNNNNNNNNPPPPII")
_GRADIENTS = struct.Struct("@PPPNNNNNNPPPNNNNNNNNN")
_ROWS = struct.Struct("@NNiPPPNNNPII")
_THREE = struct.Struct("@NNN")


def _address(buffer):
    if buffer is None:
        return 0
    if buffer.__class__ is int:
        return buffer
    try:
        return buffer.data_ptr()
    except AttributeError:
        return buffer.ptr


def _element(element: str) -> int:
    if element not in ELEMENTS:
        raise ValueError(f"element must be one of {sorted(ELEMENTS)}, not {element!r}")
    return ELEMENTS[element]


def _refused() -> hip.HipError:
    return hip.HipError(hip.INVALID_ARGUMENT, "sizes and strides are whole numbers from 0 to 2^64 - 1, "
                                              "dropped and site from 0 to 2^32 - 1")


def _packed(kind: struct.Struct, *fields) -> bytes:
    try:
        return kind.pack(*fields)
    except struct.error:
        raise _refused() from None


def _size(n) -> int:
    # A size_t argument would take what lies outside modulo 2^64.
    try:
        n = n.__index__()
    except AttributeError:
        raise _refused() from None
    if not 0 <= n < 1 << 64:
        raise _refused()
    return n


def _strides(strides, heads: int, rows: int):
    return (heads * rows * 64, rows * 64, 64) if strides is None else strides


@functools.lru_cache(maxsize=None)
def _call(name: str):
    return getattr(hip.lib(), name)


def _inputs(shape, q, k, v, element, scale, q_strides, k_strides, v_strides, query_lengths, lengths, keep, seed, site,
            dropped) -> bytes:
    _, heads, kv_heads, query_rows, rows = shape
    return _packed(_INPUTS, *shape, _element(element), scale, _address(q), _address(k), _address(v),
                   *_strides(q_strides, heads, query_rows), *_strides(k_strides, kv_heads, rows),
                   *_strides(v_strides, kv_heads, rows), _address(query_lengths), _address(lengths), _address(keep),
                   _address(seed), site, dropped)


def workspace_bytes(device: hip.Device, shape, *, element: str = "f32", backward: bool = False) -> int:
    """Bytes of workspace for `attention` (or, with backward, `attention_backward`) of exactly
    this shape and element: 0 where none is needed, and for shapes out of range, which the calls refuse."""
    try:
        return _call("irx_train_workspace_bytes")(device.handle, _packed(_SHAPE, *shape), _element(element),
                                                  bool(backward))
    except hip.HipError:
        return 0


def attention(device: hip.Device, shape, q, k, v, out, *, element: str = "f32", scale: float = 0.125, q_strides=None,
              k_strides=None, v_strides=None, out_strides=None, query_lengths=None, lengths=None, keep=None, seed=None,
              site: int = 0, dropped: int = 0, stats=None, lse=None, workspace=None, workspace_bytes: int = 0,
              stream=None) -> None:
    """D(softmax(scale q k^T)) v over the attended rows into `out`, D the weights' dropout; the
    log-sum-exp into FP32 `lse` [estimators, heads, query_rows], and what the backward pass
    needs into FP32 `stats` [estimators, heads, query_rows, 2]. 0 and -inf where a query
    attends to nothing."""
    inputs = _inputs(shape, q, k, v, element, scale, q_strides, k_strides, v_strides, query_lengths, lengths, keep, seed,
                     site, dropped)
    strides = _packed(_THREE, *_strides(out_strides, shape[1], shape[3]))
    hip.check(_call("irx_train_attention")(device.handle, inputs, _address(out), strides, _address(stats),
                                           _address(lse), _address(workspace), _size(workspace_bytes),
                                           _address(stream)))


def attention_backward(device: hip.Device, shape, q, k, v, out, stats, dout, *, dq=None, dk=None, dv=None,
                       element: str = "f32", scale: float = 0.125, q_strides=None, k_strides=None, v_strides=None,
                       out_strides=None, dout_strides=None, dq_strides=None, dk_strides=None, dv_strides=None,
                       query_lengths=None, lengths=None, keep=None, seed=None, site: int = 0, dropped: int = 0,
                       workspace=None, workspace_bytes: int = 0, stream=None) -> None:
    """The gradients of q, and of k and v, from `dout`, that of `out`; `out` and `stats` as
    `attention` wrote them with the same inputs, seed and site. Either side may be left out."""
    inputs = _inputs(shape, q, k, v, element, scale, q_strides, k_strides, v_strides, query_lengths, lengths, keep, seed,
                     site, dropped)
    _, heads, kv_heads, query_rows, rows = shape
    gradients = _packed(_GRADIENTS, _address(out), _address(stats), _address(dout),
                        *_strides(out_strides, heads, query_rows), *_strides(dout_strides, heads, query_rows),
                        _address(dq), _address(dk), _address(dv), *_strides(dq_strides, heads, query_rows),
                        *_strides(dk_strides, kv_heads, rows), *_strides(dv_strides, kv_heads, rows))
    hip.check(_call("irx_train_attention_backward")(device.handle, inputs, gradients, _address(workspace),
                                                    _size(workspace_bytes), _address(stream)))


def dropout(device: hip.Device, rows: int, width: int, x, out, *, element: str = "f32", residual=None, x_stride=None,
            residual_stride=None, out_stride=None, seed=None, site: int = 0, dropped: int = 0, stream=None) -> None:
    """residual + D(x), or D(x), of [rows, width] into `out`, which may be x or residual. Strides
    are elements from row to row, by default the width. D(gradient of out) is that of x."""
    x_stride, residual_stride, out_stride = (width if s is None else s for s in (x_stride, residual_stride, out_stride))
    hip.check(_call("irx_train_dropout")(device.handle, _packed(
        _ROWS, rows, width, _element(element), _address(x), _address(residual), _address(out), x_stride,
        residual_stride, out_stride, _address(seed), site, dropped), _address(stream)))
