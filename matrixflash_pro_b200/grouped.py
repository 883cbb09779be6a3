"""Products grouped by expert over libmfb.so (mfb_grouped_gemm / mfb_grouped_gemm_bwd_right).

The ragged form of the batch_matmul family, for the experts of a mixture-of-experts layer: the
rows of one matrix lie sorted by expert, expert e holds rows [offsets[e], offsets[e + 1]) (none
is fine), and each expert has its own weight matrix:

  grouped_matmul(left[t,k], right[e,k,n], offsets)               -> [t,n]   Y[t]  = X[t] W[e(t)]
  grouped_matmul_backward_left(grad[t,n], right[e,k,n], offsets) -> [t,k]   dX[t] = G[t] W[e(t)]^T
  grouped_matmul_backward_right(grad[t,n], left[t,k], offsets)   -> [e,k,n] dW[e] = sum_t X[t]^T G[t]

With transpose_right the weights (and their gradient) are stored [e,n,k].

Operands are float32 (strict, as GemmPrecision.fp32; tf32 permits fewer terms), float16 or
bfloat16 CUDA tensors of one type with unit stride in the last dimension; rows and matrices may be
padded or shared (strides are taken from the tensors, 0 between matrices reuses one weight). Sums
are FP32: the tensor cores add up to 512 of the contraction (strict float32: 64) with truncation,
those chunks are added with rounding, and the result is rounded once to the output's type. So the error
of the sums does not grow with their length: 5e-7 normwise for bfloat16, 7e-7 for float16 (9e-7 and 3e-6
where all products are positive), 3e-7 for strict float32, measured up to 16384 products. An infinite
float32 operand gives NaN (it has no terms to split into); those below 2^-110 lose up to 2^-134.
`out` may be given, of the operands' type or float32, and may overlap nothing that the call reads.

offsets is a contiguous int32 CUDA tensor of e + 1 entries that the kernels read: the host never
waits for group sizes, and a captured graph follows new offsets on replay. Rows in front of
offsets[0] and from offsets[e] on belong to no expert: they are 0 in a new output, left as they
were in a given `out`, and count in no gradient. Offsets that decrease or leave [0, t] are clamped
and raise InvalidArgumentError from the next sync().

The work goes to `stream`, by default the current stream of the operands' device.
"""
from __future__ import annotations

import torch

from . import _lib
from .errors import InvalidArgumentError, ShapeMismatchError
from .gemm import INT32_MAX, GemmPrecision

DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_MAX_GROUPS = 1024


# The handle of a device's current stream as an int. torch.cuda.current_stream builds a Stream object, 2 us of a
# call that takes 10 us of host time in all.
_current_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def _stream_of(device: torch.device, stream) -> int:
    return _current_raw_stream(device.index) if stream is None else stream.cuda_stream


def _new(like: torch.Tensor, shape, dtype, stream):
    """An output on `like`'s device that belongs to the stream that writes it."""
    if stream is None:
        return like.new_empty(shape, dtype=dtype)
    with torch.cuda.stream(stream):
        return like.new_empty(shape, dtype=dtype)


def _rows_ld(t: torch.Tensor, what: str, dtype) -> int:
    """Row stride of a matrix of `dtype` with unit column stride."""
    if t.dim() != 2:
        raise ShapeMismatchError(f"{what} must be a matrix")
    if t.dtype != dtype:
        raise InvalidArgumentError(f"{what} must be {dtype}")
    rows, cols = t.shape
    ld, unit = t.stride()
    if unit != 1 and cols > 1 and rows > 0:
        raise InvalidArgumentError(f"{what} must have unit column stride")
    if rows <= 1:
        return cols or 1
    if ld < cols:
        raise InvalidArgumentError(f"{what} has rows that overlap")
    return ld or 1


def _stack_ld(t: torch.Tensor, what: str, dtype, shared_ok: bool):
    """(row stride, matrix stride) of a stack of matrices of `dtype` with unit column stride."""
    if t.dim() != 3:
        raise InvalidArgumentError(f"{what} must be a rank-3 tensor")
    if t.dtype != dtype:
        raise InvalidArgumentError(f"{what} must be {dtype}")
    count, rows, cols = t.shape
    stride, ld, unit = t.stride()
    if not (count and rows and cols):
        return cols or 1, rows * cols
    if unit != 1 and cols > 1:
        raise InvalidArgumentError(f"{what} must have unit stride in its last dimension")
    if rows <= 1:
        ld = cols
    elif ld < cols:
        raise InvalidArgumentError(f"{what} has rows that overlap")
    if count <= 1:
        stride = 0 if shared_ok else rows * ld
    elif not shared_ok and stride < (rows - 1) * ld + cols:
        raise InvalidArgumentError(f"{what} has matrices that overlap")
    return ld, stride


def _check(groups: int, offsets: torch.Tensor, *tensors) -> None:
    """What both entry points ask of offsets and devices."""
    if groups > _MAX_GROUPS:
        raise InvalidArgumentError(f"at most {_MAX_GROUPS} groups are supported")
    if offsets.dtype != torch.int32 or not offsets.is_contiguous():
        raise InvalidArgumentError("offsets must be a contiguous int32 tensor")
    if offsets.dim() != 1 or offsets.shape[0] != groups + 1:
        raise ShapeMismatchError("offsets must have one entry more than there are groups")
    if not offsets.is_cuda:
        raise InvalidArgumentError("grouped products take CUDA tensors")
    device = offsets.device
    for t in tensors:
        if t is not None and t.device != device:
            raise InvalidArgumentError("operands of a grouped product must share one CUDA device")


def _dtype_of(t: torch.Tensor) -> int:
    code = DTYPES.get(t.dtype)
    if code is None:
        raise InvalidArgumentError("grouped products take float32, float16 or bfloat16 operands")
    return code


def _out_dtype(out: torch.Tensor, code: int) -> int:
    got = DTYPES.get(out.dtype)
    if got is None or (got != code and got != 0):
        raise InvalidArgumentError("out must have the operands' type or float32")
    return got


def _precision(precision) -> int:
    return 0 if precision is GemmPrecision.fp32 else int(GemmPrecision(precision))


def _launch(entry: str, what: str, device, stream, desc, offsets, a, b, out) -> None:
    status = getattr(_lib.lib(), entry)(device.index, _stream_of(device, stream), desc, offsets.data_ptr(),
                                        a.data_ptr(), b.data_ptr(), out.data_ptr())
    if status:
        _lib.check(status, what)


def _desc(*fields):
    """The descriptor; every dimension and row stride has to fit 32 bits."""
    if max(fields[:7]) > INT32_MAX:
        raise InvalidArgumentError("grouped product dimension exceeds the 32-bit limit")
    return _lib.GroupedDesc(*fields)


def _rows_times_stack(left, right, offsets, transpose, precision, out, stream, what):
    dtype = left.dtype
    code = _dtype_of(left)
    lda = _rows_ld(left, "left" if what == "grouped_matmul" else "grad", dtype)
    ldb, stride = _stack_ld(right, "right", dtype, True)
    groups, k, n = right.shape
    if transpose:
        k, n = n, k
    rows, cols = left.shape
    if cols != k:
        raise ShapeMismatchError(f"{what} shape mismatch")
    _check(groups, offsets, left, right, out)
    if out is None:
        out, out_code, ldc, rest = _new(left, (rows, n), dtype, stream), code, n or 1, 1
    else:
        if tuple(out.shape) != (rows, n):
            raise ShapeMismatchError(f"{what} output shape mismatch")
        out_code, ldc, rest = _out_dtype(out, code), _rows_ld(out, "out", out.dtype), 0
    desc = _desc(groups, rows, n, k, lda, ldb, ldc, stride, code, out_code, _precision(precision), int(transpose), rest)
    _launch("mfb_grouped_gemm", what, left.device, stream, desc, offsets, left, right, out)
    return out


def grouped_matmul(left: torch.Tensor, right: torch.Tensor, offsets: torch.Tensor, transpose_right: bool = False,
                   precision: GemmPrecision = GemmPrecision.fp32, out: torch.Tensor | None = None,
                   stream=None) -> torch.Tensor:
    """[t,k] x [e,k,n] -> [t,n]: each row times its expert's matrix ([e,n,k] with transpose_right)."""
    return _rows_times_stack(left, right, offsets, bool(transpose_right), precision, out, stream, "grouped_matmul")


def grouped_matmul_backward_left(grad: torch.Tensor, right: torch.Tensor, offsets: torch.Tensor,
                                 transpose_right: bool = False, precision: GemmPrecision = GemmPrecision.fp32,
                                 out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """dL/dleft of grouped_matmul: [t,n] x [e,k,n]^T -> [t,k]."""
    return _rows_times_stack(grad, right, offsets, not transpose_right, precision, out, stream,
                             "grouped_matmul_backward_left")


def grouped_matmul_backward_right(grad: torch.Tensor, left: torch.Tensor, offsets: torch.Tensor,
                                  transpose_right: bool = False, precision: GemmPrecision = GemmPrecision.fp32,
                                  out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """dL/dright of grouped_matmul: [e,k,n] (or [e,n,k] with transpose_right), 0 for an expert without rows."""
    what = "grouped_matmul_backward_right"
    code = _dtype_of(grad)
    a, b = (grad, left) if transpose_right else (left, grad)
    lda = _rows_ld(a, "grad" if transpose_right else "left", grad.dtype)
    ldb = _rows_ld(b, "left" if transpose_right else "grad", grad.dtype)
    if a.shape[0] != b.shape[0]:
        raise ShapeMismatchError(f"{what} shape mismatch")
    rows, k = a.shape
    n = b.shape[1]
    if offsets.dim() != 1 or offsets.shape[0] < 1:
        raise ShapeMismatchError("offsets must have one entry more than there are groups")
    groups = offsets.shape[0] - 1
    _check(groups, offsets, a, b, out)
    if out is None:
        out, out_code, ldc, stride = _new(grad, (groups, k, n), grad.dtype, stream), code, n or 1, k * n
    else:
        if tuple(out.shape) != (groups, k, n):
            raise ShapeMismatchError(f"{what} output shape mismatch")
        out_code = _out_dtype(out, code)
        ldc, stride = _stack_ld(out, "out", out.dtype, False)
    desc = _desc(groups, rows, n, k, lda, ldb, ldc, stride, code, out_code, _precision(precision), 0, 0)
    _launch("mfb_grouped_gemm_bwd_right", what, grad.device, stream, desc, offsets, a, b, out)
    return out
