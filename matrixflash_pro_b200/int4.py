"""4-bit weights over libmfb.so (mfb_quantize_int4 / mfb_dequantize_int4 / mfb_gemv_int4).

An Int4Matrix holds an n x k weight matrix (or a stack of them, one per expert) as 4-bit codes
with a scale, and optionally a zero point, per row and group of 32, 64 or 128 consecutive
columns: w = (q - z) * s, z = 8 without zero points.

  quantize_int4(weight[n,k] or [e,n,k])  -> Int4Matrix
  dequantize_int4(matrix)                -> the weights that it stands for
  gemv_int4(matrix, x[t,k])              -> [t,n]   y[r] = W x[r], for a few rows (decoding)
  gemv_int4(matrix, x[t,k], experts=ids) -> [t,n]   y[r] = W[ids[r]] x[r]

Layout, for weights from elsewhere: `packed` is a contiguous uint8 tensor [.., n, 16 * ceil(k/32)],
column j of a row in byte j // 2, even j in the low four bits, whatever is behind column k being
ignored; `scales` (float32, float16 or bfloat16) and `zeros` (uint8, 0..15) are contiguous
[.., n, ceil(k / group)].

A given `out` may overlap nothing that the call reads. The work goes to `stream`, by default the
current stream of the matrix's device.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .errors import InvalidArgumentError, ShapeMismatchError
from .gemm import checked_dim
from .grouped import DTYPES, _new, _stream_of

GEMV_ROWS = 64


class Int4Matrix:
    """A checked set of 4-bit codes, scales and zero points (layout: module text). Keeps the tensors, whose contents may
    change; which tensors they are may not, since the kernels get their addresses."""

    __slots__ = ("_packed", "_scales", "_zeros", "_k", "_group", "_n", "_experts", "_device", "_desc", "_ref")

    def __init__(self, packed: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None, k: int, group: int):
        k = checked_dim(k)
        if group not in (32, 64, 128):
            raise InvalidArgumentError("the group size of a 4-bit matrix is 32, 64 or 128")
        if packed.dtype != torch.uint8 or (zeros is not None and zeros.dtype != torch.uint8):
            raise InvalidArgumentError("packed codes and zero points must be uint8")
        if scales.dtype not in DTYPES:
            raise InvalidArgumentError("scales must be float32, float16 or bfloat16")
        if packed.dim() not in (2, 3):
            raise ShapeMismatchError("packed codes must be [n, bytes] or [experts, n, bytes]")
        if packed.shape[-1] != 16 * (-(-k // 32)):
            raise ShapeMismatchError("packed rows must take 16 * ceil(k / 32) bytes")
        want = (*packed.shape[:-1], -(-k // group))
        if tuple(scales.shape) != want or (zeros is not None and tuple(zeros.shape) != want):
            raise ShapeMismatchError("scales and zeros must be [.., n, ceil(k / group)]")
        for t in (packed, scales, zeros):
            if t is None:
                continue
            if not t.is_cuda:
                raise InvalidArgumentError("a 4-bit matrix takes CUDA tensors")
            if t.device != packed.device:
                raise InvalidArgumentError("the parts of a 4-bit matrix must share one device")
            if not t.is_contiguous():
                raise InvalidArgumentError("the parts of a 4-bit matrix must be contiguous")
        if packed.data_ptr() % 16:
            raise InvalidArgumentError("packed codes must start on a 16-byte boundary")
        self._packed, self._scales, self._zeros, self._k, self._group = packed, scales, zeros, k, int(group)
        self._n = checked_dim(packed.shape[-2])
        self._experts = checked_dim(packed.shape[0]) if packed.dim() == 3 else None
        self._device = packed.device
        self._desc = _lib.Int4MatrixDesc(packed.data_ptr(), scales.data_ptr(), 0 if zeros is None else zeros.data_ptr(),
                                         1 if self._experts is None else self._experts, self._n, k, self._group,
                                         DTYPES[scales.dtype])
        self._ref = ctypes.byref(self._desc)

    packed = property(lambda self: self._packed, doc="The codes, two a byte.")
    scales = property(lambda self: self._scales, doc="A scale per row and group.")
    zeros = property(lambda self: self._zeros, doc="A zero point per row and group, or None.")
    k = property(lambda self: self._k, doc="Columns.")
    group = property(lambda self: self._group, doc="Columns that share a scale.")
    n = property(lambda self: self._n, doc="Rows (of one matrix of a stack).")
    experts = property(lambda self: self._experts, doc="Matrices in the stack, or None for a single matrix.")
    device = property(lambda self: self._device, doc="The tensors' device.")

    @property
    def shape(self):
        """The shape of the weights that the codes stand for."""
        return torch.Size((*self._packed.shape[:-1], self._k))


def quantize_int4(weight: torch.Tensor, group: int = 128, symmetric: bool = False,
                  scale_dtype: torch.dtype | None = None, stream=None) -> Int4Matrix:
    """Codes of `weight` ([n,k] or [e,n,k], float32, float16 or bfloat16, finite). symmetric: s = max|w| / 7 and
    no zero points; else s and z span the group's range, widened to hold 0. Scales are rounded through FP32 to
    scale_dtype (default: the weight's); codes are the nearest ones, ties to even."""
    if weight.dtype not in DTYPES:
        raise InvalidArgumentError("quantize_int4 takes float32, float16 or bfloat16 weights")
    if weight.dim() not in (2, 3):
        raise ShapeMismatchError("quantize_int4 takes [n, k] or [experts, n, k] weights")
    if not weight.is_cuda:
        raise InvalidArgumentError("quantize_int4 takes CUDA tensors")
    if weight.shape[-1] > 1 and weight.numel() and weight.stride(-1) != 1:
        raise InvalidArgumentError("weight must have unit stride in its last dimension")
    if group not in (32, 64, 128):
        raise InvalidArgumentError("the group size of a 4-bit matrix is 32, 64 or 128")
    scale_dtype = weight.dtype if scale_dtype is None else scale_dtype
    if scale_dtype not in DTYPES:
        raise InvalidArgumentError("scales must be float32, float16 or bfloat16")
    *stack, n, k = weight.shape
    groups = -(-checked_dim(k) // group)
    packed = _new(weight, (*stack, n, 16 * (-(-k // 32))), torch.uint8, stream)
    scales = _new(weight, (*stack, n, groups), scale_dtype, stream)
    zeros = None if symmetric else _new(weight, (*stack, n, groups), torch.uint8, stream)
    matrix = Int4Matrix(packed, scales, zeros, k, group)
    _lib.check(_lib.lib().mfb_quantize_int4(weight.device.index, _stream_of(weight.device, stream), weight.data_ptr(),
                                            DTYPES[weight.dtype], weight.stride(-2),
                                            weight.stride(0) if stack else 0, matrix._ref), "quantize_int4")
    return matrix


def dequantize_int4(matrix: Int4Matrix, dtype: torch.dtype | None = None, out: torch.Tensor | None = None,
                    stream=None) -> torch.Tensor:
    """The weights (q - z) * s of `matrix` in FP32 (exact for 16-bit scales), rounded to `dtype` (default: the
    scales')."""
    if out is None:
        dtype = matrix.scales.dtype if dtype is None else dtype
        if dtype not in DTYPES:
            raise InvalidArgumentError("dequantize_int4 gives float32, float16 or bfloat16")
        out = _new(matrix.packed, matrix.shape, dtype, stream)
    else:
        if out.dtype not in DTYPES or (dtype is not None and dtype != out.dtype):
            raise InvalidArgumentError("out must have the asked type: float32, float16 or bfloat16")
        if out.shape != matrix.shape:
            raise ShapeMismatchError("dequantize_int4 output shape mismatch")
        if out.device != matrix.device:
            raise InvalidArgumentError("out must be on the matrix's device")
        if out.numel() and (out.stride(-1) != 1 and out.shape[-1] > 1):
            raise InvalidArgumentError("out must have unit stride in its last dimension")
        if out.shape[-2] > 1 and out.stride(-2) < out.shape[-1]:
            raise InvalidArgumentError("out has rows that overlap")
        if out.dim() == 3 and out.shape[0] > 1 and out.stride(0) < (out.shape[1] - 1) * out.stride(1) + out.shape[2]:
            raise InvalidArgumentError("out has matrices that overlap")
    _lib.check(_lib.lib().mfb_dequantize_int4(matrix.device.index, _stream_of(matrix.device, stream), matrix._ref,
                                              out.data_ptr(), DTYPES[out.dtype], out.stride(-2),
                                              out.stride(0) if out.dim() == 3 else 0), "dequantize_int4")
    return out


def gemv_int4(matrix: Int4Matrix, x: torch.Tensor, out: torch.Tensor | None = None,
              experts: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """y[r] = W x[r] for up to 64 rows of x [t,k] (float32, float16 or bfloat16); out [t,n] has x's type. A stack
    needs `experts`, a contiguous int32 CUDA tensor [t]: row r uses matrix experts[r]; a negative id gives a zero
    row, one past the stack a zero row and InvalidArgumentError from the next sync(). Sums are FP32. An infinite x
    gives the infinities (or NaN, at a weight of 0) of the formula; float32 values of x below 2^-110 lose up to 2^-134."""
    dtype, device = x.dtype, matrix._device
    code = DTYPES.get(dtype)
    if code is None:
        raise InvalidArgumentError("gemv_int4 takes float32, float16 or bfloat16 rows")
    if x.dim() != 2 or x.shape[1] != matrix._k:
        raise ShapeMismatchError("GEMV operand shape mismatch")
    if x.device != device:
        raise InvalidArgumentError("x must be on the matrix's device")
    rows = x.shape[0]
    if rows > GEMV_ROWS:
        raise InvalidArgumentError(f"gemv_int4 serves up to {GEMV_ROWS} rows (dequantize_int4 and a product serve more)")
    ldx, unit = x.stride()
    if unit != 1 and matrix._k > 1 and rows:
        raise InvalidArgumentError("x must have unit column stride")
    ids = 0
    if experts is not None:
        if experts.dtype != torch.int32 or experts.dim() != 1 or not experts.is_contiguous():
            raise InvalidArgumentError("experts must be a contiguous int32 tensor")
        if experts.shape[0] != rows:
            raise ShapeMismatchError("experts must have one entry per row")
        if experts.device != device:
            raise InvalidArgumentError("experts must be on the matrix's device")
        ids = experts.data_ptr()
    elif matrix._experts is not None:
        raise InvalidArgumentError("a stack of matrices needs an expert per row")
    n = matrix._n
    if out is None:
        out, ldy = _new(x, (rows, n), dtype, stream), n
    else:
        if out.dtype != dtype or out.device != device:
            raise InvalidArgumentError("out must have x's type and device")
        if tuple(out.shape) != (rows, n):
            raise ShapeMismatchError("GEMV operand shape mismatch")
        ldy, unit = out.stride()
        if unit != 1 and n > 1 and rows:
            raise InvalidArgumentError("out must have unit column stride")
        if rows > 1 and ldy < n:
            raise InvalidArgumentError("out has rows that overlap")
    status = _lib.lib().mfb_gemv_int4(device.index, _stream_of(device, stream), matrix._ref, rows, x.data_ptr(), ldx,
                                      code, ids, out.data_ptr(), ldy)
    if status:
        _lib.check(status, "gemv_int4")
    return out
