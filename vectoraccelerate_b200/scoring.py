"""The scoring head of an embedding model over libva_cuda: the norm that makes its queries, 4-bit tables
and their products with queries, and the loss that trains both sides.

The reference has neither of them (its int4 quantizer has one scale per array, its LogSumExp and
MatrixVector kernels work on fp32 data in memory); the classes follow the kernel classes of
``kernels.py``: constructed from a context, ``encode...`` methods over device memory, and methods that
take and return host arrays.

Device arguments are a ``DeviceBuffer``, an integer device address, or an object with ``data_ptr()``
(a torch tensor) on the context's device, laid out as documented. Work is enqueued on the context's
stream: a caller that has arrays from another stream makes that stream the context's
(``Metal4Configuration(stream=...)``) or orders the two.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass

import numpy as np

from . import _ffi
from .context import DeviceBuffer, GPUContext
from .errors import InvalidInput, raise_for_status
from .kernels import Database, TopKSelectionKernel, _f32, _Kernel

_PASS = 32  # queries that no pass over 4-bit codes exceeds (va_int4_matvec)
_ITEM = {_ffi.DTYPE_F32: 4, _ffi.DTYPE_BF16: 2, _ffi.DTYPE_INT8: 1}


class _ScoringKernel(_Kernel):
    """A kernel whose calls take device memory: keeps the device and the library's functions at hand, as a call
    for one token costs little else."""

    def __init__(self, context: GPUContext):
        super().__init__(context)
        self._device = context.device
        self._lib = _ffi.load()


def _checked(status: int, name: str) -> None:
    if status != _ffi.VA_OK:
        raise_for_status(status, f"{name}: {_ffi.last_error()}")


# Element types that a tensor may have where elements of so many bytes are expected (bf16 also as bit patterns), by
# name, and their type objects as they are met: looking an object up is what a call of a few microseconds affords.
_TYPE_NAMES = {1: {"int8", "uint8"}, 2: {"bfloat16", "int16", "uint16"}, 4: {"float32"}, 8: {"int64"}}
_TYPES = {item: set() for item in _TYPE_NAMES}


def _dense(device: int, x, count: int, item: int, name: str):
    """Device address of a contiguous array of at least ``count`` elements of ``item`` bytes; what knows its own
    size, type, device or layout is checked."""
    if x.__class__ is int:
        return x
    if x.__class__ is DeviceBuffer:
        return _buffer(device, x, count * item, name)
    try:
        if x.dtype in _TYPES[item] and x.get_device() == device and x.nbytes >= count * item and x.is_contiguous():
            return x.data_ptr()
        _check_type(x, item, name)
        if not x.is_contiguous():
            raise InvalidInput(f"{name} must be contiguous")
        if x.nbytes < count * item:
            raise InvalidInput(f"{name} holds {x.nbytes} bytes, {count * item} are needed")
        _device_of(device, x, name)
        return x.data_ptr()
    except AttributeError:
        return _buffer(device, x, 0, name)


def _strided(device: int, x, rows: int, dim: int, stride: int, item: int, name: str):
    """Device address of rows of ``dim`` elements that lie ``stride`` elements apart."""
    if x.__class__ is int:
        return x
    if x.__class__ is DeviceBuffer:
        return _buffer(device, x, ((rows - 1) * stride + dim) * item if rows > 0 else 0, name)
    try:
        if (stride == dim and x.dtype in _TYPES[item] and x.get_device() == device and x.nbytes >= rows * dim * item
                and x.is_contiguous()):
            return x.data_ptr()
        _check_type(x, item, name)
        if rows > 0 and not (stride == dim and x.is_contiguous() and x.nbytes >= rows * dim * item) and (
                x.dim() != 2 or x.shape[0] < rows or x.shape[1] < dim or (dim > 1 and x.stride(1) != 1)
                or (rows > 1 and x.stride(0) != stride)):
            raise InvalidInput(f"{name} of shape {tuple(x.shape)} and strides {x.stride()} does not hold {rows} rows of "
                               f"{dim} elements {stride} apart")
        _device_of(device, x, name)
        return x.data_ptr()
    except AttributeError:
        return _buffer(device, x, 0, name)


def _check_type(x, item: int, name: str) -> None:
    if x.itemsize != item:
        raise InvalidInput(f"{name} has elements of {x.itemsize} bytes, {item} expected")
    if str(x.dtype).rpartition(".")[2] not in _TYPE_NAMES[item]:
        raise InvalidInput(f"{name} is {x.dtype}, expected {' or '.join(sorted(_TYPE_NAMES[item]))}")
    _TYPES[item].add(x.dtype)


def _device_of(device: int, x, name: str) -> None:
    if x.get_device() != device:
        raise InvalidInput(f"{name} is on {x.device}, the context on cuda:{device}")


def _buffer(device: int, x, nbytes: int, name: str):
    if not isinstance(x, DeviceBuffer):
        raise InvalidInput(f"{name} must be a DeviceBuffer, a device address or have data_ptr(), got {type(x).__name__}")
    if x.ptr is None:
        raise InvalidInput(f"{name} has been freed")
    if x.context.device != device:
        raise InvalidInput(f"{name} is on device {x.context.device}, the context on device {device}")
    if x.nbytes < nbytes:
        raise InvalidInput(f"{name} holds {x.nbytes} bytes, {nbytes} are needed")
    return x.ptr


def _fits(**sizes) -> None:
    """Sizes that the library takes as 32-bit numbers, which the call would cut without a word."""
    for name, n in sizes.items():
        if n >> 31:
            raise InvalidInput(f"{name} must be in 0..2147483647, got {n}")


def _to_bf16(a) -> np.ndarray:
    """fp32 -> bf16 bit patterns (round to nearest even), for the host-array methods."""
    u = np.ascontiguousarray(a, np.float32).view(np.uint32)
    nan = (u & 0x7FFFFFFF) > 0x7F800000
    r = ((u + np.uint32(0x7FFF) + ((u >> np.uint32(16)) & np.uint32(1))) >> np.uint32(16)).astype(np.uint16)
    return np.where(nan, ((u >> np.uint32(16)) | np.uint32(0x40)).astype(np.uint16), r)


def _whole(a, dtype, name: str) -> np.ndarray:
    """Host array of whole numbers as ``dtype``, which has to hold them."""
    a = np.asarray(a)
    if a.size and (a.dtype.kind not in "iu" or int(a.min()) < np.iinfo(dtype).min or int(a.max()) > np.iinfo(dtype).max):
        raise InvalidInput(f"{name} must be whole numbers that {np.dtype(dtype)} holds, got {a.dtype}")
    return np.ascontiguousarray(a, dtype)


def _from_bf16(b) -> np.ndarray:
    return (np.ascontiguousarray(b, np.uint16).astype(np.uint32) << np.uint32(16)).view(np.float32)


def int4_row_bytes(dimension: int) -> int:
    """Bytes of a coded row (VA_INT4_ROW_BYTES)."""
    return (dimension + 31) // 32 * 16


class RMSNormInt8Kernel(_ScoringKernel):
    """Root-mean-square norm with the residual's addition and int8 codes with scales (va_rms_norm_int8)."""

    def encode(self, x, weight, rows: int, dimension: int, codes, scales, residual=None, residual_out=None,
               dtype: int = _ffi.DTYPE_BF16, epsilon: float = 1e-6, group: int = 0, x_stride: int | None = None,
               residual_stride: int | None = None) -> None:
        """codes [rows x dimension] int8 and scales [rows x groups] fp32 (one group per row when ``group`` is 0) of
        h = x + residual; ``residual_out`` receives h. Strides in elements; the dimension by default."""
        if dtype not in (_ffi.DTYPE_F32, _ffi.DTYPE_BF16):
            raise InvalidInput(f"dtype must be DTYPE_F32 or DTYPE_BF16, got {dtype}")
        if (dimension | group) >> 31:
            _fits(dimension=dimension, group=group)
        dev, item = self._device, _ITEM[dtype]
        xs = dimension if x_stride is None else x_stride
        rs = dimension if residual_stride is None else residual_stride
        groups = -(-dimension // group) if group > 0 else 1
        n = rows * dimension
        _checked(self._lib.va_rms_norm_int8(
            self.context.handle, _strided(dev, x, rows, dimension, xs, item, "x"),
            None if residual is None else _strided(dev, residual, rows, dimension, rs, item, "residual"),
            _dense(dev, weight, dimension, item, "weight"), rows, dimension, dtype, xs, rs, epsilon, group,
            None if residual_out is None else _dense(dev, residual_out, n, item, "residual_out"),
            _dense(dev, codes, n, 1, "codes"), _dense(dev, scales, rows * groups, 4, "scales")), "va_rms_norm_int8")

    def compute(self, x, weight, residual=None, epsilon: float = 1e-6, group: int = 0):
        """fp32 host arrays -> (codes int8 [rows, dim], scales [rows, groups], h [rows, dim])."""
        a, w = _f32(x), np.ascontiguousarray(weight, np.float32)
        rows, dim = a.shape
        if w.shape != (dim,):
            raise InvalidInput(f"weight must have {dim} elements, got shape {w.shape}")
        ctx = self.context
        r = None
        if residual is not None:
            r = _f32(residual)
            if r.shape != a.shape:
                raise InvalidInput(f"residual shape {r.shape} differs from {a.shape}")
        groups = -(-dim // group) if group > 0 else 1
        dx, dw = ctx.get_buffer_for(a), ctx.get_buffer_for(w)
        dr = ctx.get_buffer_for(r) if r is not None else None
        codes = ctx.get_buffer(rows * dim, np.int8, (rows, dim))
        scales = ctx.get_buffer(4 * rows * groups, np.float32, (rows, groups))
        self.encode(dx, dw, rows, dim, codes, scales, dr, dr, _ffi.DTYPE_F32, epsilon, group)
        return codes.download(), scales.download(), dr.download() if dr is not None else a


@dataclass
class Int4Rows:
    """4-bit rows in device memory: codes [n x int4_row_bytes(dim)], scales and zero points [n x groups]."""

    codes: DeviceBuffer
    scales: DeviceBuffer
    zero_points: DeviceBuffer | None
    n: int
    dim: int
    group: int
    scale_dtype: int


class Int4GroupQuantizationKernel(_ScoringKernel):
    """4-bit codes with a scale, and optionally a zero point, per group of 32, 64 or 128 columns
    (va_sq_quantize_int4_groups; the codes' format is ScalarQuantizationKernel's)."""

    def encode(self, x, rows: int, dimension: int, group: int, codes, scales, zero_points=None,
               dtype: int = _ffi.DTYPE_F32, scale_dtype: int = _ffi.DTYPE_BF16, x_stride: int | None = None) -> None:
        _check_types(dtype, scale_dtype, group, (_ffi.DTYPE_F32, _ffi.DTYPE_BF16))
        if dimension >> 31:
            _fits(dimension=dimension)
        dev = self._device
        stride = dimension if x_stride is None else x_stride
        groups = -(-dimension // group)
        _checked(self._lib.va_sq_quantize_int4_groups(
            self.context.handle, _strided(dev, x, rows, dimension, stride, _ITEM[dtype], "x"), dtype, rows, dimension, stride,
            group, scale_dtype, _dense(dev, codes, rows * int4_row_bytes(dimension), 1, "codes"),
            _dense(dev, scales, rows * groups, _ITEM[scale_dtype], "scales"),
            None if zero_points is None else _dense(dev, zero_points, rows * groups, 1, "zero_points")),
            "va_sq_quantize_int4_groups")

    def quantize(self, rows, group: int = 64, type: str = "symmetric",  # noqa: A002
                 scale_dtype: int = _ffi.DTYPE_BF16) -> Int4Rows:
        """Codes of fp32 host rows."""
        a = _f32(rows)
        if a.size == 0:
            raise InvalidInput("Empty input")
        if type not in ("symmetric", "asymmetric"):
            raise InvalidInput(f"type must be 'symmetric' or 'asymmetric', got {type!r}")
        _check_types(_ffi.DTYPE_F32, scale_dtype, group, (_ffi.DTYPE_F32,))
        n, dim = a.shape
        groups = -(-dim // group)
        ctx = self.context
        codes = ctx.get_buffer(n * int4_row_bytes(dim), np.uint8, (n, int4_row_bytes(dim)))
        scales = ctx.get_buffer(n * groups * _ITEM[scale_dtype],
                                np.uint16 if scale_dtype == _ffi.DTYPE_BF16 else np.float32, (n, groups))
        zeros = ctx.get_buffer(n * groups, np.int8, (n, groups)) if type == "asymmetric" else None
        dx = ctx.get_buffer_for(a)
        self.encode(dx, n, dim, group, codes, scales, zeros, _ffi.DTYPE_F32, scale_dtype)
        ctx.synchronize()
        return Int4Rows(codes, scales, zeros, n, dim, group, scale_dtype)

    def dequantize(self, rows: Int4Rows) -> np.ndarray:
        """The fp32 values that the codes stand for."""
        ctx = self.context
        out = ctx.get_buffer(4 * rows.n * rows.dim, np.float32, (rows.n, rows.dim))
        groups = -(-rows.dim // rows.group)
        _ffi.call("va_sq_dequantize_int4_groups", self._h,
                  _dense(self._device, rows.codes, rows.n * int4_row_bytes(rows.dim), 1, "codes"),
                  _dense(self._device, rows.scales, rows.n * groups, _ITEM[rows.scale_dtype], "scales"),
                  None if rows.zero_points is None else _dense(self._device, rows.zero_points, rows.n * groups, 1, "zero_points"),
                  rows.n, rows.dim, rows.group, rows.scale_dtype, out.ptr)
        return out.download()


def _check_types(dtype: int, scale_dtype: int, group: int, dtypes) -> None:
    if dtype not in dtypes:
        raise InvalidInput(f"dtype must be one of {dtypes}, got {dtype}")
    if scale_dtype not in (_ffi.DTYPE_F32, _ffi.DTYPE_BF16):
        raise InvalidInput(f"scale_dtype must be DTYPE_F32 or DTYPE_BF16, got {scale_dtype}")
    if group not in (32, 64, 128):
        raise InvalidInput(f"group must be 32, 64 or 128, got {group}")


class Int4MatVecKernel(_ScoringKernel):
    """Products of a few queries with 4-bit rows (va_int4_matvec): fp32 scores [queries x rows]."""

    def encode(self, queries, num_queries: int, codes, scales, rows: int, dimension: int, group: int, out,
               zero_points=None, query_dtype: int = _ffi.DTYPE_F32, query_scales=None,
               scale_dtype: int = _ffi.DTYPE_BF16, out_stride: int | None = None) -> None:
        """Queries [num_queries x dimension] contiguous, of ``query_dtype``; int8 queries take a scale each from
        ``query_scales``."""
        _check_types(query_dtype, scale_dtype, group, _ITEM)
        if (dimension | num_queries) >> 31:
            _fits(dimension=dimension, num_queries=num_queries)
        dev = self._device
        stride = rows if out_stride is None else out_stride
        groups = -(-dimension // group)
        _checked(self._lib.va_int4_matvec(
            self.context.handle, _dense(dev, queries, num_queries * dimension, _ITEM[query_dtype], "queries"), query_dtype,
            None if query_scales is None else _dense(dev, query_scales, num_queries, 4, "query_scales"), num_queries,
            _dense(dev, codes, rows * int4_row_bytes(dimension), 1, "codes"),
            _dense(dev, scales, rows * groups, _ITEM[scale_dtype], "scales"),
            None if zero_points is None else _dense(dev, zero_points, rows * groups, 1, "zero_points"), rows, dimension, group,
            scale_dtype, _strided(dev, out, num_queries, rows, stride, 4, "out"), stride), "va_int4_matvec")

    def compute(self, queries, table: Int4Rows) -> np.ndarray:
        """fp32 host queries -> scores [queries, rows]."""
        q = _f32(queries)
        if q.shape[1] != table.dim:
            raise InvalidInput(f"query dimension {q.shape[1]} != table dimension {table.dim}")
        ctx = self.context
        dq = ctx.get_buffer_for(q)
        out = ctx.get_buffer(4 * q.shape[0] * table.n, np.float32, (q.shape[0], table.n))
        self.encode(dq, q.shape[0], table.codes, table.scales, table.n, table.dim, table.group, out, table.zero_points,
                    _ffi.DTYPE_F32, None, table.scale_dtype)
        return out.download()


class Int4Database:
    """Resident 4-bit rows searched by inner product: scores of every row (Int4MatVecKernel), then the
    k largest (TopKSelectionKernel's selection), ids by (score, id). The fp32 rows are not kept."""

    SCORE_BYTES = 1 << 28  # of scores that a search keeps at a time (at least those of 32 queries)

    def __init__(self, context: GPUContext, rows, group: int = 64, type: str = "symmetric",  # noqa: A002
                 scale_dtype: int = _ffi.DTYPE_BF16):
        self.context = context
        self.table = Int4GroupQuantizationKernel(context).quantize(rows, group, type, scale_dtype)
        self.n, self.dim = self.table.n, self.table.dim
        self._matvec = Int4MatVecKernel(context)

    def scores(self, queries) -> np.ndarray:
        return self._matvec.compute(queries, self.table)

    def search(self, queries, k: int, query_scales=None):
        """-> (values [Q, k], ids [Q, k]). Queries are fp32, or int8 codes with a scale per query (the output of
        RMSNormInt8Kernel)."""
        int8 = query_scales is not None
        q = _whole(queries, np.int8, "queries with query_scales") if int8 else np.ascontiguousarray(queries, np.float32)
        if q.ndim == 1:
            q = q[None, :]
        if q.shape[1] != self.dim:
            raise InvalidInput(f"query dimension {q.shape[1]} != database dimension {self.dim}")
        if not 0 < k <= TopKSelectionKernel.maxK:
            raise InvalidInput(f"K must be between 1 and {TopKSelectionKernel.maxK}")
        ctx, t, nq = self.context, self.table, q.shape[0]
        ds = None
        if int8:
            s = np.ascontiguousarray(query_scales, np.float32).ravel()
            if s.shape != (nq,):
                raise InvalidInput(f"query_scales must have one entry per query ({nq}), got {s.size}")
            ds = ctx.get_buffer_for(s)
        dq = ctx.get_buffer_for(q)
        # Scores of so many queries at a time as SCORE_BYTES hold, a multiple of what a pass over the codes takes.
        chunk = max(1, min(nq, max(_PASS, self.SCORE_BYTES // (4 * self.n) // _PASS * _PASS)))
        scores = ctx.get_buffer(4 * chunk * self.n, np.float32, (chunk, self.n))
        vals, ids = ctx.get_buffer(4 * nq * k, np.float32, (nq, k)), ctx.get_buffer(4 * nq * k, np.uint32, (nq, k))
        for q0 in range(0, nq, chunk):
            count = min(chunk, nq - q0)
            self._matvec.encode(dq.ptr + q0 * self.dim * q.itemsize, count, t.codes, t.scales, self.n, self.dim, t.group, scores,
                                t.zero_points, _ffi.DTYPE_INT8 if int8 else _ffi.DTYPE_F32, ds.ptr + 4 * q0 if int8 else None,
                                t.scale_dtype)
            _ffi.call("va_topk_select", ctx.handle, scores.ptr, count, self.n, self.n, k, _ffi.SELECT_MAX, vals.ptr + 4 * q0 * k,
                      ids.ptr + 4 * q0 * k, k)
        return vals.download(), ids.download()

    def close(self) -> None:
        for b in (self.table.codes, self.table.scales, self.table.zero_points):
            if b is not None:
                b.free()


class SoftmaxCrossEntropyKernel(_ScoringKernel):
    """Softmax cross entropy of tokens against all rows of a table, logits never kept, with the gradients
    of both sides (va_softmax_xent_forward / _backward). The table is bf16: device memory or a bf16
    ``Database``."""

    def workspace_bytes(self, tokens: int, rows: int, dimension: int, backward: bool) -> int:
        _fits(dimension=dimension)
        n = ctypes.c_size_t()
        _ffi.call("va_softmax_xent_workspace", self._h, tokens, rows, dimension, int(backward), ctypes.byref(n))
        return n.value

    def _table(self, table, rows: int, dimension: int, stride: int):
        if isinstance(table, Database):
            if table.context.device != self._device:
                raise InvalidInput(f"table is on device {table.context.device}, the context on device {self._device}")
            if table.dtype != _ffi.DTYPE_BF16 or table.dim != dimension or stride != dimension or table.n < rows:
                raise InvalidInput(f"table must be a bf16 database of at least {rows} rows x {dimension}")
            return table.rows_ptr()
        return _strided(self._device, table, rows, dimension, stride, 2, "table")

    def _workspace(self, workspace, tokens, rows, dimension, backward):
        if workspace is None:
            return None, 0
        if isinstance(workspace, int):
            at, nbytes = workspace, self.workspace_bytes(tokens, rows, dimension, backward)
        elif not hasattr(workspace, "data_ptr"):
            at, nbytes = _buffer(self._device, workspace, 0, "workspace"), workspace.nbytes
        else:
            _device_of(self._device, workspace, "workspace")
            if not workspace.is_contiguous():
                raise InvalidInput("workspace must be contiguous")
            at, nbytes = workspace.data_ptr(), workspace.nbytes
        if not at and tokens > 0:  # (address 0 would stand for the context's scratch)
            raise InvalidInput("workspace of 0 bytes is too small")
        return at, nbytes

    def encode_forward(self, hidden, table, labels, tokens: int, rows: int, dimension: int, loss, lse,
                       logit_scale: float = 1.0, hidden_stride: int | None = None, table_stride: int | None = None,
                       workspace=None) -> None:
        """hidden [tokens x dimension], table [rows x dimension] bf16; labels int64 (outside [0, rows): no
        loss); loss and lse [tokens] fp32. An integer ``workspace`` address must hold workspace_bytes()."""
        if dimension >> 31:
            _fits(dimension=dimension)
        dev = self._device
        hs = dimension if hidden_stride is None else hidden_stride
        ts = dimension if table_stride is None else table_stride
        ws, nbytes = self._workspace(workspace, tokens, rows, dimension, False)
        _checked(self._lib.va_softmax_xent_forward(
            self.context.handle, _strided(dev, hidden, tokens, dimension, hs, 2, "hidden"), hs,
            self._table(table, rows, dimension, ts), ts, _dense(dev, labels, tokens, 8, "labels"), tokens, rows, dimension,
            logit_scale, ws, nbytes, _dense(dev, loss, tokens, 4, "loss"), _dense(dev, lse, tokens, 4, "lse")),
            "va_softmax_xent_forward")

    def encode_backward(self, hidden, table, labels, lse, grad_loss, tokens: int, rows: int, dimension: int, grad_hidden,
                        grad_table, logit_scale: float = 1.0, hidden_stride: int | None = None,
                        table_stride: int | None = None, workspace=None) -> None:
        """Gradients of sum(grad_loss * loss) (``grad_loss`` None: 1), bf16 and contiguous, written whole."""
        if dimension >> 31:
            _fits(dimension=dimension)
        dev = self._device
        hs = dimension if hidden_stride is None else hidden_stride
        ts = dimension if table_stride is None else table_stride
        ws, nbytes = self._workspace(workspace, tokens, rows, dimension, True)
        _checked(self._lib.va_softmax_xent_backward(
            self.context.handle, _strided(dev, hidden, tokens, dimension, hs, 2, "hidden"), hs,
            self._table(table, rows, dimension, ts), ts, _dense(dev, labels, tokens, 8, "labels"),
            _dense(dev, lse, tokens, 4, "lse"), None if grad_loss is None else _dense(dev, grad_loss, tokens, 4, "grad_loss"),
            tokens, rows, dimension, logit_scale, ws, nbytes, _dense(dev, grad_hidden, tokens * dimension, 2, "grad_hidden"),
            _dense(dev, grad_table, rows * dimension, 2, "grad_table")), "va_softmax_xent_backward")

    def compute(self, hidden, table, labels, logit_scale: float = 1.0, grad_loss=None):
        """Host arrays (hidden and table are rounded to bf16) -> (loss [T], lse [T], grad_hidden [T, D],
        grad_table [V, D]), fp32."""
        h, w = _to_bf16(_f32(hidden)), _to_bf16(_f32(table))
        y = _whole(labels, np.int64, "labels").ravel()
        if h.shape[1] != w.shape[1]:
            raise InvalidInput("Dimension mismatch in input vectors")
        if y.shape != (h.shape[0],):
            raise InvalidInput(f"labels must have one entry per token ({h.shape[0]}), got {y.size}")
        t, v, d = h.shape[0], w.shape[0], h.shape[1]
        ctx = self.context
        dh, dw, dy = ctx.get_buffer_for(h), ctx.get_buffer_for(w), ctx.get_buffer_for(y)
        loss, lse = ctx.get_buffer(4 * t, np.float32, (t,)), ctx.get_buffer(4 * t, np.float32, (t,))
        gh, gw = ctx.get_buffer(2 * t * d, np.uint16, (t, d)), ctx.get_buffer(2 * v * d, np.uint16, (v, d))
        dg = None
        if grad_loss is not None:
            g = np.ascontiguousarray(grad_loss, np.float32).ravel()
            if g.shape != (t,):
                raise InvalidInput(f"grad_loss must have one entry per token ({t}), got {g.size}")
            dg = ctx.get_buffer_for(g)
        self.encode_forward(dh, dw, dy, t, v, d, loss, lse, logit_scale)
        self.encode_backward(dh, dw, dy, lse, dg, t, v, d, gh, gw, logit_scale)
        return loss.download(), lse.download(), _from_bf16(gh.download()), _from_bf16(gw.download())
