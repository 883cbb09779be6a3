"""CPU tier: what the 4-bit weights refuse, before any launch, in Python and through the C ABI."""
import ctypes

import pytest
import torch

import matrixflash_pro_b200 as mf
from matrixflash_pro_b200 import _lib


def test_host_tensors_are_rejected():
    with pytest.raises(mf.InvalidArgumentError):
        mf.quantize_int4(torch.ones(4, 64))
    with pytest.raises(mf.InvalidArgumentError):
        mf.Int4Matrix(torch.zeros(4, 32, dtype=torch.uint8), torch.ones(4, 1), None, 64, 64)


@pytest.mark.parametrize("packed,scales,zeros,k,group,error", [
    ((4, 32), (4, 2), None, 64, 48, mf.InvalidArgumentError),
    ((4, 31), (4, 2), None, 64, 32, mf.ShapeMismatchError),
    ((4, 32), (4, 1), None, 64, 32, mf.ShapeMismatchError),
    ((4, 32), (4, 2), (4, 1), 64, 32, mf.ShapeMismatchError),
    ((32,), (2,), None, 64, 32, mf.ShapeMismatchError),
    ((4, 48), (4, 2), None, 64, 32, mf.ShapeMismatchError),
    ((2, 4, 32), (4, 2), None, 64, 32, mf.ShapeMismatchError),
])
def test_matrix_shapes(packed, scales, zeros, k, group, error):
    with pytest.raises(error):
        mf.Int4Matrix(torch.zeros(packed, dtype=torch.uint8), torch.ones(scales),
                      None if zeros is None else torch.zeros(zeros, dtype=torch.uint8), k, group)


def test_matrix_types():
    ok = torch.zeros(4, 32, dtype=torch.uint8)
    with pytest.raises(mf.InvalidArgumentError):
        mf.Int4Matrix(ok.int(), torch.ones(4, 2), None, 64, 32)
    with pytest.raises(mf.InvalidArgumentError):
        mf.Int4Matrix(ok, torch.ones(4, 2).double(), None, 64, 32)
    with pytest.raises(mf.InvalidArgumentError):
        mf.Int4Matrix(ok, torch.ones(4, 2), torch.ones(4, 2), 64, 32)
    for bad in (torch.ones(4, 64).double(), torch.ones(4, 64).int()):
        with pytest.raises(mf.InvalidArgumentError):
            mf.quantize_int4(bad)
    with pytest.raises(mf.ShapeMismatchError):
        mf.quantize_int4(torch.ones(64))


P, S, Z, X, Y = 0x100000, 0x200000, 0x300000, 0x400000, 0x500000


def _matrix(**kw):
    base = dict(packed=P, scales=S, zeros=Z, experts=1, n=4, k=64, group=32, scale_dtype=0)
    base.update(kw)
    return _lib.Int4MatrixDesc(*(base[f] for f, _ in _lib.Int4MatrixDesc._fields_))


@pytest.mark.parametrize("kw,needle", [
    (dict(experts=-1), "non-negative"), (dict(n=-1), "non-negative"), (dict(k=-1), "non-negative"),
    (dict(group=16), "group"), (dict(scale_dtype=3), "scale type"), (dict(packed=0), "null"), (dict(scales=0), "null"),
    (dict(packed=P + 8), "16-byte"), (dict(scales=S + 2), "aligned"),
])
def test_abi_rejects_matrices(kw, needle):
    lib = mf.lib()
    m = ctypes.byref(_matrix(**kw))
    for st in (lib.mfb_quantize_int4(0, None, X, 0, 64, 0, m), lib.mfb_dequantize_int4(0, None, m, X, 0, 64, 0),
               lib.mfb_gemv_int4(0, None, m, 1, X, 64, 0, 0, Y, 4)):
        assert st == _lib.MFB_EINVAL and needle in _lib.last_error()


def test_abi_rejects_operands():
    lib = mf.lib()
    m = ctypes.byref(_matrix())
    stack = ctypes.byref(_matrix(experts=3))

    def refused(st, needle):
        assert st == _lib.MFB_EINVAL and needle in _lib.last_error()

    refused(lib.mfb_gemv_int4(0, None, None, 1, X, 64, 0, 0, Y, 4), "null")
    refused(lib.mfb_gemv_int4(0, None, m, -1, X, 64, 0, 0, Y, 4), "rows")
    refused(lib.mfb_gemv_int4(0, None, m, 65, X, 64, 0, 0, Y, 4), "rows")
    refused(lib.mfb_gemv_int4(0, None, stack, 1, X, 64, 0, 0, Y, 4), "expert")
    refused(lib.mfb_gemv_int4(0, None, m, 2, X, 64, 0, 0, Y, 3), "stride")
    refused(lib.mfb_gemv_int4(0, None, m, 1, X, 64, 7, 0, Y, 4), "type")
    refused(lib.mfb_gemv_int4(0, None, m, 1, 0, 64, 0, 0, Y, 4), "null")
    refused(lib.mfb_gemv_int4(0, None, m, 1, X + 2, 64, 0, 0, Y, 4), "aligned")
    refused(lib.mfb_gemv_int4(0, None, m, 1, X, 64, 0, 0, X + 16, 4), "alias")
    refused(lib.mfb_dequantize_int4(0, None, m, X, 0, 63, 0), "stride")
    refused(lib.mfb_dequantize_int4(0, None, stack, X, 0, 64, 255), "stride")
    refused(lib.mfb_dequantize_int4(0, None, m, 0, 0, 64, 0), "null")
    refused(lib.mfb_quantize_int4(0, None, X + 1, 1, 64, 0, m), "aligned")
    assert lib.mfb_gemv_int4(0, None, m, 0, 0, 0, 0, 0, 0, 0) == _lib.MFB_OK
    assert lib.mfb_dequantize_int4(0, None, ctypes.byref(_matrix(n=0)), 0, 0, 0, 0) == _lib.MFB_OK


@pytest.mark.parametrize("at", [P, P + 4 * 32 - 4, S, S + 4 * 2 * 4 - 4, Z, Z + 4, P - 12])
def test_abi_rejects_outputs_over_the_matrix(at):
    # 4 rows of 64 codes, 2 scales and 2 zero points; y takes 16 bytes, the weights 1024
    lib = mf.lib()
    m = ctypes.byref(_matrix())
    for st in (lib.mfb_gemv_int4(0, None, m, 1, X, 64, 0, 0, at, 4), lib.mfb_dequantize_int4(0, None, m, at, 0, 64, 0),
               lib.mfb_quantize_int4(0, None, at, 0, 64, 0, m)):
        assert st == _lib.MFB_EINVAL and "alias" in _lib.last_error()
    assert lib.mfb_gemv_int4(0, None, m, 1, X, 64, 0, Y + 12, Y, 4) == _lib.MFB_EINVAL
    assert "alias" in _lib.last_error()
    assert lib.mfb_gemv_int4(0, None, m, 1, X, 64, 0, Y + 66, Y, 4) == _lib.MFB_EINVAL
    assert "aligned" in _lib.last_error()


@pytest.mark.parametrize("name", ["packed", "scales", "zeros", "k", "group", "n", "experts", "device", "shape"])
def test_the_parts_of_a_matrix_cannot_be_exchanged(name):
    """The kernels get addresses that were taken when the matrix was made."""
    matrix = object.__new__(mf.Int4Matrix)
    with pytest.raises(AttributeError):
        setattr(matrix, name, None)
