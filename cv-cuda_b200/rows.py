"""Row operators: LayerNorm and the embedding lookup, each with its gradient, on torch CUDA tensors.

They sit between what the image operators produce (normalised batches, patches, label maps and the token ids that come with
them) and the first activations of a model: :func:`layernorm` is the sibling of :func:`cvcuda_b200.normalize` that takes the
statistics from the data, :func:`embedding` the sibling of :func:`cvcuda_b200.convertto` that gathers. The reference has no
counterpart. PyTorch provides memory and streams; every value is computed by ``libcvcuda_b200.so`` through
``include/cvcuda_b200/row_ops.h``.

The functions do not take part in torch's autograd: gradients are calls of their own (``layernorm_backward``,
``embedding_backward``). A tensor may be CUDA memory of any device (the call runs there) or page-locked host memory. Outputs and
workspaces are allocated on the stream the call runs on; on a ``stream`` other than torch's current one, the caller orders the
two as for every other operator here.
"""
from __future__ import annotations

import contextlib
import ctypes as C
import math
import struct
from functools import lru_cache
from typing import Optional, Tuple

import torch

from . import ops
from .ops import Error, Status, _check


class _Rows(C.Structure):
    _fields_ = [("base", C.c_void_p), ("dtype", C.c_int32), ("cols", C.c_int64), ("count", C.c_int64 * 3), ("stride", C.c_int64 * 3)]


class _LayerNormOp(C.Structure):
    _fields_ = [("weight", C.c_void_p), ("bias", C.c_void_p), ("weightType", C.c_int32), ("biasType", C.c_int32),
                ("epsilon", C.c_float), ("mean", C.c_void_p), ("rstd", C.c_void_p)]


class _LayerNormGradOp(C.Structure):
    _fields_ = [("mean", C.c_void_p), ("rstd", C.c_void_p), ("weight", C.c_void_p), ("weightType", C.c_int32),
                ("dweight", C.c_void_p), ("dbias", C.c_void_p), ("dweightType", C.c_int32), ("dbiasType", C.c_int32)]


class _EmbeddingGradOp(C.Structure):
    _fields_ = [("scale", C.c_float), ("accumulate", C.c_int32), ("paddingIndex", C.c_int64)]


_TYPES = {torch.uint8: 0, torch.float32: 6, torch.float16: 7, torch.bfloat16: 8, torch.int32: 5, torch.int64: 9}
_FLOATS = (torch.float32, torch.float16, torch.bfloat16)

# the current device, and the handle of its current stream without building a Stream object, where this torch has them
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", lambda device: torch.cuda.current_stream(device).cuda_stream)


@lru_cache(maxsize=None)
def _cuda(device: int) -> torch.device:
    return torch.device("cuda", device)


_bound: Optional[C.CDLL] = None


def _lib() -> C.CDLL:
    global _bound
    L = ops.lib()
    if _bound is not L:
        R = S = O = C.c_void_p
        for name, args in (("LayerNormWorkspace", [R, S]),
                           ("LayerNorm", [R, R, O, C.c_void_p, C.c_size_t, C.c_void_p]),
                           ("LayerNormBackwardWorkspace", [R, S]),
                           ("LayerNormBackward", [R, R, R, O, C.c_void_p, C.c_size_t, C.c_void_p]),
                           ("Embedding", [R, R, R, C.c_float, C.c_void_p]),
                           ("EmbeddingBackwardWorkspace", [R, R, S]),
                           ("EmbeddingBackward", [R, R, R, O, C.c_void_p, C.c_size_t, C.c_void_p])):
            f = getattr(L, "b200pp" + name)
            f.restype, f.argtypes = C.c_int, args
        _bound = L
    return _bound


# ------------------------------------------------------------------------------------------------ arguments

def _invalid(message: str) -> Error:
    return Error(Status.ERROR_INVALID_ARGUMENT, message)


def _device_of(first, *others) -> int:
    """Index of the device the call runs on: that of the CUDA tensors, which must agree (page-locked host tensors follow)."""
    try:
        dev = first.get_device() if first.is_cuda else _host(first)
        for t in others:
            if t is not None:
                d = t.get_device() if t.is_cuda else _host(t)
                if d != dev:
                    if dev < 0:
                        dev = d
                    elif d >= 0:
                        raise _invalid(f"Tensors are on different devices (cuda:{dev} and cuda:{d})")
    except AttributeError:
        raise _invalid("Arguments must be cuda-accessible, pitch-linear tensors") from None
    return dev if dev >= 0 else torch.cuda.current_device()


def _host(t) -> int:
    if not t.is_pinned():
        raise _invalid("Arguments must be cuda-accessible, pitch-linear tensors")
    return -1


def _view(t: torch.Tensor, axes: int, what: str):
    """(columns, [(count, stride in elements)]): the rows the last `axes` dimensions of `t` make, in the order of the others,
    dimensions that continue one another merged."""
    shape, lead = t.shape, t.dim() - axes
    cols = 1
    for k in range(lead, lead + axes):
        cols *= shape[k]
    if t.is_contiguous():
        return cols, ((t.numel() // cols if cols else math.prod(shape[:lead]), cols),)
    stride = t.stride()
    step = 1
    for k in range(t.dim() - 1, lead - 1, -1):
        if stride[k] != step and shape[k] != 1:
            raise _invalid(f"{what}: the last {axes} dimension(s) must be contiguous")
        step *= shape[k]
    dims = []
    for k in range(lead):
        n, s = shape[k], stride[k]
        if n == 1:
            continue
        if dims and dims[-1][1] == n * s:
            dims[-1] = (dims[-1][0] * n, s)
        else:
            dims.append((n, s))
    if len(dims) > 3:
        raise _invalid(f"{what} has more than three independently strided dimensions of rows")
    return cols, dims


# The C structures as bytes, which ctypes passes by address: a third of the time a ctypes.Structure takes to fill in.
_pack_rows = struct.Struct("=Qi4xq3q3q").pack
_pack_ln = struct.Struct("=QQiif4xQQ").pack
_pack_ln_grad = struct.Struct("=QQQi4xQQii").pack
_pack_emb_grad = struct.Struct("=fiq").pack
_pack_float = struct.Struct("=f").pack
assert struct.calcsize("=Qi4xq3q3q") == C.sizeof(_Rows) and struct.calcsize("=QQiif4xQQ") == C.sizeof(_LayerNormOp)
assert struct.calcsize("=QQQi4xQQii") == C.sizeof(_LayerNormGradOp) and struct.calcsize("=fiq") == C.sizeof(_EmbeddingGradOp)


def _rows(t: torch.Tensor, axes: int, what: str):
    """(B200ppRows as bytes, columns, rows)."""
    cols, dims = _view(t, axes, what)
    es = t.element_size()
    code = _TYPES.get(t.dtype, -1)
    if len(dims) == 1:
        n, s = dims[0]
        return _pack_rows(t.data_ptr(), code, cols, n, 1, 1, s * es, 0, 0), cols, n
    c, d, rows = [1, 1, 1], [0, 0, 0], 1
    for k, (n, s) in enumerate(dims):
        c[k], d[k] = n, s * es
        rows *= n
    return _pack_rows(t.data_ptr(), code, cols, *c, *d), cols, rows


def _axes_of(t: torch.Tensor, axes: int) -> int:
    axes = int(axes)
    if axes < 1 or axes > t.dim():
        raise _invalid(f"axes must be 1 to {t.dim()} for a tensor of {t.dim()} dimension(s)")
    return axes


def _param(t: torch.Tensor, numel: int, what: str, kinds=_FLOATS) -> Tuple[int, int]:
    """(address, type code) of a packed tensor of `numel` values."""
    if t.dtype not in kinds:
        raise _invalid(f"Invalid DataType of the {what}")
    if t.numel() != numel or not t.is_contiguous():
        raise _invalid(f"The {what} must be packed and hold {numel} value(s)")
    return t.data_ptr(), _TYPES[t.dtype]


_NOT_FLOAT32 = (struct.error, OverflowError)  # what packing raises for anything but a number that float32 holds


def _enter(device: int, stream):
    """(handle of the launch stream, what to leave afterwards or None). Makes the device and the stream torch's current ones where
    they are not, so that what the call allocates belongs to that stream."""
    current = _raw_stream(device)
    handle = current if stream is None else ops._stream_handle(stream)
    other = device != _current_device()
    if not other and handle == current:
        return handle, None
    stack = contextlib.ExitStack()
    if other:
        stack.enter_context(torch.cuda.device(device))
    if handle != current:
        if not isinstance(stream, torch.cuda.Stream):
            stream = torch.cuda.ExternalStream(handle, device=device) if handle else torch.cuda.default_stream(device)
        elif stream.device.index != device:
            stack.close()
            raise _invalid(f"The stream belongs to {stream.device}, the tensors to cuda:{device}")
        stack.enter_context(torch.cuda.stream(stream))
    return handle, stack


@lru_cache(maxsize=1024)
def _workspace_size(name: str, code: int, cols: int, rows: int) -> int:
    """What the library asks for; it depends on the shape alone."""
    n = C.c_size_t(0)
    _check(getattr(_lib(), name)(_pack_rows(256, code, cols, rows, 1, 1, cols * 8, 0, 0), C.byref(n)))
    return n.value


@lru_cache(maxsize=1024)
def _embedding_workspace_size(code: int, cols: int, count: int, dcode: int, rows: int) -> int:
    n = C.c_size_t(0)
    _check(_lib().b200ppEmbeddingBackwardWorkspace(_pack_rows(256, code, cols, count, 1, 1, cols * 8, 0, 0),
                                                   _pack_rows(256, dcode, cols, rows, 1, 1, cols * 8, 0, 0), C.byref(n)))
    return n.value


def _scratch(size: int, device: int) -> torch.Tensor:
    return torch.empty_strided((size,), (1,), dtype=torch.uint8, device=_cuda(device))


def _like(t: torch.Tensor, kind: torch.dtype, device: int) -> torch.Tensor:
    """A packed tensor of the shape of `t` on the device (empty_like takes half of the time of empty, but keeps strides)."""
    if t.is_cuda and t.is_contiguous():
        return torch.empty_like(t, dtype=kind)
    return torch.empty(t.shape, dtype=kind, device=_cuda(device))


# ------------------------------------------------------------------------------------------------ LayerNorm

_WHOLE_ROWS = 8192  # rows up to this length need no workspace (row_ops.h)


def _layernorm(d, src, weight, bias, epsilon, axes, mean, rstd, device, handle):
    """`d`: the output, as _rows packs it, or the tensor `src` is laid out like, freshly allocated."""
    s, cols, count = _rows(src, axes, "Input")
    if not isinstance(d, bytes):
        d = _pack_rows(d.data_ptr(), _TYPES.get(d.dtype, -1), cols, count, 1, 1, cols * d.element_size(), 0, 0)
    w, wt = _param(weight, cols, "weight") if weight is not None else (0, 0)
    b, bt = _param(bias, cols, "bias") if bias is not None else (0, 0)
    m = _param(mean, count, "mean", (torch.float32,))[0] if mean is not None else 0
    r = _param(rstd, count, "rstd", (torch.float32,))[0] if rstd is not None else 0
    try:
        op = _pack_ln(w, b, wt, bt, epsilon, m, r)
    except _NOT_FLOAT32:
        raise _invalid("epsilon must be a float32 number") from None
    keep, ws, size = None, None, 0
    if cols > _WHOLE_ROWS:
        size = _workspace_size("b200ppLayerNormWorkspace", _TYPES.get(src.dtype, -1), cols, count)
        keep = _scratch(size, device)
        ws = keep.data_ptr()
    _check(_lib().b200ppLayerNorm(s, d, op, ws, size, handle))


def layernorm_into(dst: torch.Tensor, src: torch.Tensor, weight: Optional[torch.Tensor] = None,
                   bias: Optional[torch.Tensor] = None, epsilon: float = 1e-5, *, axes: int = 1,
                   mean: Optional[torch.Tensor] = None, rstd: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """LayerNorm into ``dst`` (float16, bfloat16 or float32, the shape of ``src``): see :func:`layernorm`. ``mean`` and
    ``rstd``: packed float32 tensors, one value per row, that receive the statistics. ``dst`` may be ``src``."""
    device = _device_of(src, dst, weight, bias, mean, rstd)
    axes = _axes_of(src, axes)
    if dst.shape != src.shape:
        raise _invalid("Input and output shapes are different")
    handle, leave = _enter(device, stream)
    try:
        _layernorm(_rows(dst, axes, "Output")[0], src, weight, bias, epsilon, axes, mean, rstd, device, handle)
    finally:
        if leave is not None:
            leave.close()
    return dst


def layernorm(src: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
              epsilon: float = 1e-5, *, axes: int = 1, data_type: Optional[torch.dtype] = None, stats: bool = False, stream=None):
    """``(src - mean) / sqrt(variance + epsilon) * weight + bias`` with the mean and variance of each row, a row being the last
    ``axes`` dimensions of ``src``: 1 normalises the channels of an NHWC tensor or the features of tokens, 3 whole HWC images
    (per-image standardisation). ``src``: uint8, float16, bfloat16 or float32; the dimensions of a row must be contiguous, the
    others may have any strides. ``weight`` / ``bias``: one value per element of a row, or None. The result has
    ``data_type`` (float16, bfloat16 or float32; default: that of ``src``, float32 for uint8). With ``stats``, returns
    (result, mean, rstd), the float32 statistics of the rows that :func:`layernorm_backward` takes."""
    device = _device_of(src, weight, bias)
    axes = _axes_of(src, axes)
    kind = data_type or (src.dtype if src.dtype != torch.uint8 else torch.float32)
    handle, leave = _enter(device, stream)
    try:
        dst = _like(src, kind, device)
        mean = rstd = None
        if stats:
            mean = torch.empty(src.shape[:src.dim() - axes], dtype=torch.float32, device=_cuda(device))
            rstd = torch.empty_like(mean)
        _layernorm(dst, src, weight, bias, epsilon, axes, mean, rstd, device, handle)
    finally:
        if leave is not None:
            leave.close()
    return (dst, mean, rstd) if stats else dst


def _layernorm_backward(d, dweight, dbias, grad, src, mean, rstd, weight, axes, device, handle):
    s, cols, count = _rows(src, axes, "Input")
    g = _rows(grad, axes, "Gradient")[0]
    if d is not None and not isinstance(d, bytes):
        d = _pack_rows(d.data_ptr(), _TYPES.get(d.dtype, -1), cols, count, 1, 1, cols * d.element_size(), 0, 0)
    w, wt = _param(weight, cols, "weight") if weight is not None else (0, 0)
    dw, dwt = _param(dweight, cols, "weight gradient") if dweight is not None else (0, 0)
    db, dbt = _param(dbias, cols, "bias gradient") if dbias is not None else (0, 0)
    op = _pack_ln_grad(_param(mean, count, "mean", (torch.float32,))[0], _param(rstd, count, "rstd", (torch.float32,))[0], w, wt,
                       dw, db, dwt, dbt)
    keep, ws, size = None, None, 0
    if dw or db:
        size = _workspace_size("b200ppLayerNormBackwardWorkspace", _TYPES.get(src.dtype, -1), cols, count)
        if size:
            keep = _scratch(size, device)
            ws = keep.data_ptr()
    _check(_lib().b200ppLayerNormBackward(g, s, d, op, ws, size, handle))


def layernorm_backward_into(dsrc: Optional[torch.Tensor], dweight: Optional[torch.Tensor], dbias: Optional[torch.Tensor],
                            grad: torch.Tensor, src: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor,
                            weight: Optional[torch.Tensor] = None, *, axes: int = 1, stream=None):
    """The gradients of :func:`layernorm` into the tensors given (None: not wanted): see :func:`layernorm_backward`.
    ``dsrc`` may be ``grad`` or ``src``."""
    device = _device_of(grad, src, mean, rstd, weight, dsrc, dweight, dbias)
    axes = _axes_of(src, axes)
    if grad.shape != src.shape or (dsrc is not None and dsrc.shape != src.shape):
        raise _invalid("Input and gradient shapes are different")
    handle, leave = _enter(device, stream)
    try:
        _layernorm_backward(None if dsrc is None else _rows(dsrc, axes, "Input gradient")[0], dweight, dbias, grad, src, mean, rstd,
                            weight, axes, device, handle)
    finally:
        if leave is not None:
            leave.close()
    return dsrc, dweight, dbias


def layernorm_backward(grad: torch.Tensor, src: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor,
                       weight: Optional[torch.Tensor] = None, *, axes: int = 1, data_type: Optional[torch.dtype] = None,
                       src_grad: bool = True, weight_grad: bool = True, bias_grad: bool = True, stream=None):
    """(dsrc, dweight, dbias): the gradients of :func:`layernorm`, given that of its result and the statistics it returned;
    None for those switched off. ``dsrc`` has ``data_type`` (default: the type of ``src``, that of ``grad`` for uint8);
    ``dweight`` and ``dbias`` have the type of ``weight`` (float32 without one) and the shape of a row."""
    device = _device_of(grad, src, mean, rstd, weight)
    axes = _axes_of(src, axes)
    if grad.shape != src.shape:
        raise _invalid("Input and gradient shapes are different")
    handle, leave = _enter(device, stream)
    try:
        dsrc = dweight = dbias = None
        if src_grad:
            dsrc = _like(src, data_type or (src.dtype if src.dtype != torch.uint8 else grad.dtype), device)
        if weight_grad or bias_grad:
            row = src.shape[src.dim() - axes:]
            if weight is not None and weight.shape == row:
                one = lambda: _like(weight, weight.dtype, device)  # noqa: E731
            else:
                kind = weight.dtype if weight is not None else torch.float32
                one = lambda: torch.empty(row, dtype=kind, device=_cuda(device))  # noqa: E731
            dweight = one() if weight_grad else None
            dbias = one() if bias_grad else None
        _layernorm_backward(dsrc, dweight, dbias, grad, src, mean, rstd, weight, axes, device, handle)
    finally:
        if leave is not None:
            leave.close()
    return dsrc, dweight, dbias


# ------------------------------------------------------------------------------------------------ embedding lookup

def _indices(indices: torch.Tensor) -> bytes:
    return _rows(indices, 0, "Indices")[0]


def embedding_into(dst: torch.Tensor, indices: torch.Tensor, table: torch.Tensor, scale: float = 1.0, *, stream=None) -> torch.Tensor:
    """Embedding lookup into ``dst`` (the shape of ``indices`` followed by the number of columns): see :func:`embedding`."""
    device = _device_of(table, indices, dst)
    if table.dim() != 2 or dst.shape != (*indices.shape, table.shape[1]):
        raise _invalid("The output must have the indices' shape followed by the table's number of columns")
    handle, leave = _enter(device, stream)
    try:
        _pack_float(scale)
        _check(_lib().b200ppEmbedding(_indices(indices), _rows(table, 1, "Table")[0], _rows(dst, 1, "Output")[0], scale, handle))
    except _NOT_FLOAT32:
        raise _invalid("The scale must be a float32 number") from None
    finally:
        if leave is not None:
            leave.close()
    return dst


def embedding(indices: torch.Tensor, table: torch.Tensor, scale: float = 1.0, *, data_type: Optional[torch.dtype] = None,
              stream=None) -> torch.Tensor:
    """``scale * table[indices]``: ``indices`` (uint8, int32 or int64, any shape) select rows of ``table`` [rows, columns]
    (float16, bfloat16 or float32) -- tokens, positions, class labels, the colours of a label map. An index outside the table
    gives zeros. The result has ``data_type`` (default: that of ``table``)."""
    device = _device_of(table, indices)
    if table.dim() != 2:
        raise _invalid("Table must have two dimensions")
    handle, leave = _enter(device, stream)
    try:
        i, _, count = _rows(indices, 0, "Indices")
        t, cols, _ = _rows(table, 1, "Table")
        shape = (*indices.shape, cols)
        if table.is_cuda:
            dst = table.new_empty(shape, dtype=data_type)
        else:
            dst = torch.empty(shape, dtype=data_type or table.dtype, device=_cuda(device))
        d = _pack_rows(dst.data_ptr(), _TYPES.get(dst.dtype, -1), cols, count, 1, 1, cols * dst.element_size(), 0, 0)
        _pack_float(scale)
        _check(_lib().b200ppEmbedding(i, t, d, scale, handle))
    except _NOT_FLOAT32:
        raise _invalid("The scale must be a float32 number") from None
    finally:
        if leave is not None:
            leave.close()
    return dst


def _embedding_backward(dtable, grad, indices, scale, padding_index, accumulate, device, handle):
    g, cols, count = _rows(grad, 1, "Gradient")
    t, _, rows = _rows(dtable, 1, "Table gradient")
    if padding_index is None or not 0 <= padding_index < rows:
        padding_index = -1
    try:
        op = _pack_emb_grad(scale, int(accumulate), int(padding_index))
    except _NOT_FLOAT32:
        raise _invalid("The scale must be a float32 number") from None
    size = _embedding_workspace_size(_TYPES.get(grad.dtype, -1), cols, count, _TYPES.get(dtable.dtype, -1), rows)
    keep = _scratch(size, device) if size else None
    _check(_lib().b200ppEmbeddingBackward(g, _indices(indices), t, op, keep.data_ptr() if size else None, size, handle))


def embedding_backward_into(dtable: torch.Tensor, grad: torch.Tensor, indices: torch.Tensor, scale: float = 1.0, *,
                            padding_index: Optional[int] = None, accumulate: bool = False, stream=None) -> torch.Tensor:
    """The gradient of :func:`embedding` with respect to the table into ``dtable``, or added to it with ``accumulate``
    (rows no index names are then left alone): see :func:`embedding_backward`."""
    device = _device_of(dtable, grad, indices)
    if dtable.dim() != 2 or grad.shape != (*indices.shape, dtable.shape[1]):
        raise _invalid("The gradient must have the indices' shape followed by the table's number of columns")
    handle, leave = _enter(device, stream)
    try:
        _embedding_backward(dtable, grad, indices, scale, padding_index, accumulate, device, handle)
    finally:
        if leave is not None:
            leave.close()
    return dtable


def embedding_backward(grad: torch.Tensor, indices: torch.Tensor, rows: int, scale: float = 1.0, *,
                       padding_index: Optional[int] = None, data_type: torch.dtype = torch.float32, stream=None) -> torch.Tensor:
    """The gradient of :func:`embedding` with respect to a table of ``rows`` rows: row v is ``scale`` times the sum of the rows
    of ``grad`` whose index is v, zero if there is none. Indices outside the table and those equal to ``padding_index`` take
    no part. The sums are float32, in an order that the indices, the types and the tensors' layout settle, rounded to ``data_type``
    once."""
    device = _device_of(grad, indices)
    if grad.dim() < 1 or grad.shape[:-1] != indices.shape:
        raise _invalid("The gradient must have the indices' shape followed by the table's number of columns")
    rows = int(rows)
    if rows < 0:
        raise _invalid("The table must not have a negative number of rows")
    handle, leave = _enter(device, stream)
    try:
        dtable = torch.empty((rows, grad.shape[-1]), dtype=data_type, device=_cuda(device))
        _embedding_backward(dtable, grad, indices, scale, padding_index, False, device, handle)
    finally:
        if leave is not None:
            leave.close()
    return dtable


__all__ = ["layernorm", "layernorm_into", "layernorm_backward", "layernorm_backward_into", "embedding", "embedding_into",
           "embedding_backward", "embedding_backward_into"]
