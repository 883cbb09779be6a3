"""CPU tier: what the grouped products refuse, before any launch, in Python and through the C ABI."""
import ctypes

import pytest
import torch

import matrixflash_pro_b200 as mf
from matrixflash_pro_b200 import _lib

OFF = torch.tensor([0, 1, 3], dtype=torch.int32)


def test_host_tensors_are_rejected():
    with pytest.raises(mf.InvalidArgumentError):
        mf.grouped_matmul(torch.ones(3, 4), torch.ones(2, 4, 5), OFF)
    with pytest.raises(mf.InvalidArgumentError):
        mf.grouped_matmul_backward_left(torch.ones(3, 5), torch.ones(2, 4, 5), OFF)
    with pytest.raises(mf.InvalidArgumentError):
        mf.grouped_matmul_backward_right(torch.ones(3, 5), torch.ones(3, 4), OFF)


@pytest.mark.parametrize("left,right,off,error", [
    (torch.ones(3), torch.ones(2, 4, 5), OFF, mf.ShapeMismatchError),
    (torch.ones(3, 4), torch.ones(4, 5), OFF, mf.InvalidArgumentError),
    (torch.ones(3, 6), torch.ones(2, 4, 5), OFF, mf.ShapeMismatchError),
    (torch.ones(3, 4).half(), torch.ones(2, 4, 5), OFF, mf.InvalidArgumentError),
    (torch.ones(3, 4).int(), torch.ones(2, 4, 5).int(), OFF, mf.InvalidArgumentError),
    (torch.ones(4, 3).t(), torch.ones(2, 4, 5), OFF, mf.InvalidArgumentError),
    (torch.ones(1, 4).expand(3, 4), torch.ones(2, 4, 5), OFF, mf.InvalidArgumentError),
    (torch.ones(3, 4), torch.ones(2, 5, 4).transpose(1, 2), OFF, mf.InvalidArgumentError),
    (torch.ones(3, 4), torch.ones(2, 4, 5), OFF.long(), mf.InvalidArgumentError),
    (torch.ones(3, 4), torch.ones(2, 4, 5), OFF[:2], mf.ShapeMismatchError),
    (torch.ones(3, 4), torch.ones(2, 4, 5), torch.zeros(6, dtype=torch.int32)[::2], mf.InvalidArgumentError),
])
def test_shapes_types_and_strides(left, right, off, error):
    with pytest.raises(error):
        mf.grouped_matmul(left, right, off)


def test_backward_right_refusals():
    with pytest.raises(mf.ShapeMismatchError):
        mf.grouped_matmul_backward_right(torch.ones(3, 5), torch.ones(4, 4), OFF)
    with pytest.raises(mf.ShapeMismatchError):
        mf.grouped_matmul_backward_right(torch.ones(3, 5), torch.ones(3, 4), torch.zeros(0, dtype=torch.int32))
    with pytest.raises(mf.InvalidArgumentError):
        mf.grouped_matmul_backward_right(torch.ones(3, 5), torch.ones(3, 4).half(), OFF)


def _desc(**kw):
    base = dict(groups=2, rows=3, n=5, k=4, lda=4, ldb=5, ldc=5, stride=20, dtype=0, out_dtype=0, precision=0,
                trans_b=0, zero_rest=0)
    base.update(kw)
    return _lib.GroupedDesc(*(base[f] for f, _ in _lib.GroupedDesc._fields_))


A, B, C, O = 0x100000, 0x200000, 0x300000, 0x400000


@pytest.mark.parametrize("kw,needle", [
    (dict(groups=-1), "non-negative"), (dict(rows=-1), "non-negative"), (dict(n=-2), "non-negative"),
    (dict(groups=1025), "1024"), (dict(dtype=3), "type"), (dict(dtype=1, out_dtype=2), "type"),
    (dict(precision=2), "precision"), (dict(trans_b=2), "trans_b"), (dict(zero_rest=-1), "zero_rest"),
    (dict(lda=3), "lda"), (dict(ldb=4), "ldb"), (dict(trans_b=1, ldb=3), "ldb"), (dict(ldc=4), "ldc"),
    (dict(stride=-1), "stride"),
])
def test_abi_rejects_descriptors(kw, needle):
    st = mf.lib().mfb_grouped_gemm(0, None, ctypes.byref(_desc(**kw)), O, A, B, C)
    assert st == _lib.MFB_EINVAL and needle in _lib.last_error()


def test_abi_rejects_pointers_and_aliases():
    lib = mf.lib()
    d = _desc()
    for args, needle in (((0, A, B, C), "offsets"), ((O, 0, B, C), "null"), ((O, A, 0, C), "null"),
                         ((O, A, B, 0), "null"), ((O, A, B, A + 40), "alias"), ((O, A, B, B + 156), "alias"),
                         ((O, A + 2, B, C), "aligned")):
        assert lib.mfb_grouped_gemm(0, None, ctypes.byref(d), *args) == _lib.MFB_EINVAL
        assert needle in _lib.last_error()
    assert lib.mfb_grouped_gemm(0, None, None, O, A, B, C) == _lib.MFB_EINVAL
    right = lib.mfb_grouped_gemm_bwd_right
    assert right(0, None, ctypes.byref(_desc(stride=19)), O, A, B, C) == _lib.MFB_EINVAL
    assert "overlap" in _lib.last_error()
    assert right(0, None, ctypes.byref(_desc(trans_b=1)), O, A, B, C) == _lib.MFB_EINVAL
    assert right(0, None, ctypes.byref(_desc(zero_rest=1)), O, A, B, C) == _lib.MFB_EINVAL
    # an output that only the last group reaches into
    assert right(0, None, ctypes.byref(_desc()), O, A, B, A - 100) == _lib.MFB_EINVAL
    assert "alias" in _lib.last_error()
    # nothing to do needs no device
    assert lib.mfb_grouped_gemm(0, None, ctypes.byref(_desc(rows=0)), O, 0, 0, 0) == _lib.MFB_OK
    assert right(0, None, ctypes.byref(_desc(groups=0)), O, 0, 0, 0) == _lib.MFB_OK


def test_abi_rejects_outputs_over_the_offsets():
    lib = mf.lib()
    for entry in (lib.mfb_grouped_gemm, lib.mfb_grouped_gemm_bwd_right):
        for offsets, needle in ((C, "alias"), (C + 4, "alias"), (C - 4, "alias"), (C - 4096 + 2, "aligned")):
            assert entry(0, None, ctypes.byref(_desc()), offsets, A, B, C) == _lib.MFB_EINVAL
            assert needle in _lib.last_error()


@pytest.mark.parametrize("kw", [dict(k=0, lda=1), dict(groups=0), dict(rows=0)])
def test_abi_rejects_misaligned_outputs_of_calls_that_read_nothing(kw):
    """Such calls still write zeros (rows of no group, empty sums)."""
    lib = mf.lib()
    entry = lib.mfb_grouped_gemm_bwd_right if "rows" in kw else lib.mfb_grouped_gemm
    for c, types in ((C + 2, {}), (C + 1, dict(dtype=2, out_dtype=2)), (C + 2, dict(dtype=1))):
        st = entry(0, None, ctypes.byref(_desc(**kw, **types)), O, A, B, c)
        assert st == _lib.MFB_EINVAL and "aligned" in _lib.last_error()
