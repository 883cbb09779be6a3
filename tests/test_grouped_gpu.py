"""GPU tier: products grouped by expert against FP64 products of the same operands.

Tolerance, elementwise: |y - y64| <= u (k / 8 + 32) S + r |y64|, S = sum |a_i b_i| in FP64. u = 2^-23 (the tensor
cores add with truncation), k / 8 counts two additions per 16 of k; the 32 stands for what does not grow with k:
the two terms of an FP32 product that strict mode leaves out (below 2^-21) and the last additions. r is half a
step of a 16-bit output, 0 for FP32. Strict FP32 also holds the library's normwise 1e-6. TF32: S * 2^-13 more
(two BF16 terms, the first one cut and the second one rounded, leave at most 2^-15 of each factor, and the product of
the second terms, at most 2^-14, is left out)."""
import pytest
import torch

import matrixflash_pro_b200 as mf
from helpers import STRICT_NORMWISE

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = 2.0 ** -23


def _normal(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def _offsets(sizes, first=0):
    ends = [first]
    for s in sizes:
        ends.append(ends[-1] + s)
    return torch.tensor(ends, dtype=torch.int32, device="cuda")


def _reference(a, b, offsets, out=None):
    """(y64, S) with y64 = out's rows (or 0) outside the groups; b as [e, k, n]."""
    n = b.shape[2]
    y = torch.zeros(a.shape[0], n, dtype=torch.float64, device="cuda") if out is None else out.double()
    s = torch.zeros(a.shape[0], n, dtype=torch.float64, device="cuda")
    o = offsets.tolist()
    for e in range(len(o) - 1):
        rows = slice(o[e], o[e + 1])
        x, w = a[rows].double(), b[e].double()
        y[rows] = x @ w
        s[rows] = x.abs() @ w.abs()
    return y, s


def _reference_right(a, b, offsets):
    o = offsets.tolist()
    y = torch.zeros(len(o) - 1, a.shape[1], b.shape[1], dtype=torch.float64, device="cuda")
    s = torch.zeros_like(y)
    for e in range(len(o) - 1):
        x, g = a[o[e]:o[e + 1]].double(), b[o[e]:o[e + 1]].double()
        y[e] = x.T @ g
        s[e] = x.abs().T @ g.abs()
    return y, s


def _bound(y, s, k, dtype, tf32=False):
    half_step = 0.0 if dtype == F32 else torch.finfo(dtype).eps / 2
    smallest = 0.0 if dtype == F32 else torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    return U * (k / 8 + 32) * s + half_step * y.abs() + smallest + (2.0 ** -13 * s if tf32 else 0.0)


def _check(got, y, s, k, tf32=False):
    mf.sync()
    err = (got.double() - y).abs()
    over = err - _bound(y, s, k, got.dtype, tf32)
    assert torch.isfinite(got).all()
    assert (over <= 0).all(), f"worst {err.max().item():.3e}, over by {over.max().item():.3e}"
    if got.dtype == F32 and not tf32 and y.norm() > 0:
        assert ((got.double() - y).norm() / y.norm()).item() <= STRICT_NORMWISE


SIZES = [
    [1], [0], [5, 0, 1], [128, 256, 64], [0, 0, 7, 0], [33, 65, 129, 257, 1, 0, 2], [300, 0, 511, 16, 17, 31, 32],
    [1] * 40,
]
SHAPES = [(64, 128), (256, 256), (1, 1), (17, 3), (130, 250), (72, 520), (1000, 40), (65, 1024)]


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("i", range(len(SIZES)))
def test_forward_and_backward(dtype, trans, i):
    sizes = SIZES[i]
    for j, (k, n) in enumerate(SHAPES if i in (5, 6) else SHAPES[i % 3::3]):
        off = _offsets(sizes)
        rows, e = sum(sizes), len(sizes)
        seed = 100 * i + j
        x, g = _normal((rows, k), dtype, seed), _normal((rows, n), dtype, seed + 1)
        w = _normal((e, n, k) if trans else (e, k, n), dtype, seed + 2, k ** -0.5)
        b = w.transpose(1, 2) if trans else w
        _check(mf.grouped_matmul(x, w, off, trans), *_reference(x, b, off), k)
        _check(mf.grouped_matmul_backward_left(g, w, off, trans), *_reference(g, b.transpose(1, 2), off), n)
        y, s = _reference_right(x, g, off)
        got = mf.grouped_matmul_backward_right(g, x, off, trans)
        _check(got.transpose(1, 2) if trans else got, y, s, rows)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("k,n", [(2048, 512), (768, 2048), (4097, 129)])
def test_longer_sums_and_ragged_groups(dtype, k, n):
    sizes = [700, 0, 13, 256, 1, 511, 90]
    off = _offsets(sizes)
    x, g = _normal((sum(sizes), k), dtype, 1), _normal((sum(sizes), n), dtype, 2)
    w = _normal((len(sizes), k, n), dtype, 3, k ** -0.5)
    _check(mf.grouped_matmul(x, w, off), *_reference(x, w, off), k)
    _check(mf.grouped_matmul_backward_left(g, w, off), *_reference(g, w.transpose(1, 2), off), n)
    _check(mf.grouped_matmul_backward_right(g, x, off), *_reference_right(x, g, off), sum(sizes))


def test_same_sign_sums_are_not_biased():
    """All products positive: what truncation drops adds up, and strict FP32 still holds 1e-6."""
    x = _normal((200, 4096), F32, 1).abs()
    w = _normal((2, 4096, 130), F32, 2).abs()
    off = _offsets([150, 50])
    _check(mf.grouped_matmul(x, w, off), *_reference(x, w, off), 4096)
    g = _normal((4096, 70), F32, 3).abs()
    a = _normal((4096, 96), F32, 4).abs()
    off = _offsets([1, 4095])
    _check(mf.grouped_matmul_backward_right(g, a, off), *_reference_right(a, g, off), 4096)


def test_values_over_the_whole_fp32_range():
    """Factors of very different size, exact powers and the largest finite values."""
    x = torch.ldexp(_normal((64, 40), F32, 1), torch.randint(-30, 30, (64, 40), device="cuda").int())
    w = torch.ldexp(_normal((1, 40, 48), F32, 2), torch.randint(-30, 30, (1, 40, 48), device="cuda").int())
    off = _offsets([64])
    y, s = _reference(x, w, off)
    got = mf.grouped_matmul(x, w, off)
    mf.sync()
    assert ((got.double() - y).abs() <= _bound(y, s, 40, F32)).all()
    big = torch.full((3, 1), 3.4028234e38, device="cuda")
    one = torch.tensor([[[1.0, 0.5, -0.25]]], device="cuda")
    got = mf.grouped_matmul(big, one, _offsets([3]))
    mf.sync()
    assert torch.equal(got, big * one[0])


@pytest.mark.parametrize("trans", [False, True])
def test_tf32_permits_fewer_terms(trans):
    sizes, k, n = [100, 3, 0, 260], 500, 300
    off = _offsets(sizes)
    x, g = _normal((363, k), F32, 1), _normal((363, n), F32, 2)
    w = _normal((4, n, k) if trans else (4, k, n), F32, 3)
    b = w.transpose(1, 2) if trans else w
    tf32 = mf.GemmPrecision.tf32
    _check(mf.grouped_matmul(x, w, off, trans, tf32), *_reference(x, b, off), k, True)
    _check(mf.grouped_matmul_backward_left(g, w, off, trans, tf32), *_reference(g, b.transpose(1, 2), off), n, True)
    _check(mf.grouped_matmul_backward_right(g, x, off, False, tf32), *_reference_right(x, g, off), 363, True)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_rows_outside_the_groups(dtype):
    """Rows in front of the first and behind the last group: NaN there reaches nothing, a new output has zeros, a
    given one keeps what it holds."""
    k, n, sizes = 72, 136, [5, 0, 40]
    off = _offsets(sizes, first=3)
    rows = 3 + 45 + 70
    x, g, w = _normal((rows, k), dtype, 1), _normal((rows, n), dtype, 2), _normal((3, k, n), dtype, 3)
    for t in (x, g):
        t[:3] = float("nan")
        t[48:] = float("nan")
    inside = slice(3, 48)
    _check(mf.grouped_matmul(x, w, off), *_reference(x, w, off), k)
    out = torch.full((rows, n), 7.0, dtype=dtype, device="cuda")
    assert mf.grouped_matmul(x, w, off, out=out) is out
    y, s = _reference(x, w, off, torch.full_like(out, 7.0))
    _check(out, y, s, k)
    assert (out[:3] == 7).all() and (out[48:] == 7).all() and (out[inside] != 7).any()
    _check(mf.grouped_matmul_backward_left(g, w, off), *_reference(g, w.transpose(1, 2), off), n)
    _check(mf.grouped_matmul_backward_right(g, x, off), *_reference_right(x, g, off), 45)


@pytest.mark.parametrize("dtype", [F32, F16], ids=str)
def test_nan_stays_in_its_group(dtype):
    sizes = [37, 50, 29]
    off = _offsets(sizes)
    x, g, w = _normal((116, 96), dtype, 1), _normal((116, 80), dtype, 2), _normal((3, 96, 80), dtype, 3)
    clean = mf.grouped_matmul(x, w, off), mf.grouped_matmul_backward_right(g, x, off)
    x[40, 7] = float("nan")
    x[60] = float("inf")
    g[41, 3] = float("-inf")
    y, d = mf.grouped_matmul(x, w, off), mf.grouped_matmul_backward_right(g, x, off)
    mf.sync()
    keep = torch.ones(116, dtype=torch.bool, device="cuda")
    keep[40] = keep[60] = False
    assert torch.equal(y[keep], clean[0][keep]) and y[40].isnan().all() and not y[60].isfinite().any()
    assert torch.equal(d[0], clean[1][0]) and torch.equal(d[2], clean[1][2])
    assert d[1][7].isnan().all()


def test_empty_calls():
    off = _offsets([0, 0])
    w = _normal((2, 8, 16), BF16, 1)
    assert mf.grouped_matmul(w.new_empty((0, 8)), w, off).shape == (0, 16)
    d = mf.grouped_matmul_backward_right(w.new_empty((0, 16)), w.new_empty((0, 8)), off)
    y = mf.grouped_matmul(w.new_ones((4, 8)), w, off)  # four rows of no expert
    z = mf.grouped_matmul(w.new_ones((4, 0)), w.new_empty((2, 0, 5)), _offsets([1, 3]))  # k = 0
    none = mf.grouped_matmul(w.new_ones((4, 8)), w[:0], _offsets([]))
    mf.sync()
    assert d.shape == (2, 8, 16) and not d.any() and not y.any() and z.shape == (4, 5) and not z.any()
    assert none.shape == (4, 16) and not none.any()
    assert mf.grouped_matmul(w.new_ones((4, 8)), w.new_empty((2, 8, 0)), off).shape == (4, 0)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=str)
def test_strides_and_offset_bases(dtype):
    """Padded rows, columns cut out of wider rows (any element address), shared weights, every third matrix."""
    sizes, k, n = [20, 70, 0, 3], 88, 104
    off = _offsets(sizes)
    for cut in (0, 1, 8):
        x = _normal((93, k + 24), dtype, 1)[:, cut:cut + k]
        g = _normal((93, n + 9), dtype, 2)[:, cut:cut + n]
        w = _normal((12, k + 3, n + 16), dtype, 3)[::3, 3:, cut:cut + n]
        _check(mf.grouped_matmul(x, w, off), *_reference(x, w, off), k)
        _check(mf.grouped_matmul_backward_left(g, w, off), *_reference(g, w.transpose(1, 2), off), n)
        _check(mf.grouped_matmul_backward_right(g, x, off), *_reference_right(x, g, off), 93)
        _check(mf.grouped_matmul_backward_right(g, x, off, True).transpose(1, 2), *_reference_right(x, g, off), 93)
    shared = _normal((1, k, n), dtype, 4).expand(4, k, n)
    _check(mf.grouped_matmul(x, shared, off), *_reference(x, shared, off), k)
    wide = torch.full((4, k, n + 5), 3.0, dtype=dtype, device="cuda")
    y, s = _reference_right(x, g, off)
    _check(mf.grouped_matmul_backward_right(g, x, off, out=wide[:, :, 2:2 + n]), y, s, 93)
    assert (wide[:, :, :2] == 3).all() and (wide[:, :, 2 + n:] == 3).all()
    out = torch.full((93, n + 3), 3.0, dtype=dtype, device="cuda")
    _check(mf.grouped_matmul(x, w, off, out=out[:, 1:n + 1]), *_reference(x, w, off), k)
    assert (out[:, 0] == 3).all() and (out[:, n + 1:] == 3).all()


@pytest.mark.parametrize("dtype", [F16, BF16], ids=str)
def test_fp32_output_of_16_bit_operands(dtype):
    sizes, k, n = [40, 260, 5], 320, 144
    off = _offsets(sizes)
    x, g, w = _normal((305, k), dtype, 1), _normal((305, n), dtype, 2), _normal((3, k, n), dtype, 3)
    out = torch.empty(305, n, device="cuda")
    _check(mf.grouped_matmul(x, w, off, out=out), *_reference(x, w, off), k, True)
    dw = torch.empty(3, k, n, device="cuda")
    _check(mf.grouped_matmul_backward_right(g, x, off, out=dw), *_reference_right(x, g, off), 305, True)
    # and no further off than their FP32 sums are
    y, s = _reference(x, w, off)
    assert ((out.double() - y).abs() <= U * (k / 8 + 32) * s).all()


def test_positions_past_32_bits():
    """Rows and matrices more than 2^31 elements from the start of their tensor."""
    ld = 3 << 28
    base = torch.empty(2 * ld + 64, dtype=BF16, device="cuda")
    x = base.as_strided((3, 64), (ld, 1))
    x.copy_(_normal((3, 64), BF16, 1))
    w = _normal((2, 64, 96), BF16, 2)
    off = _offsets([1, 2])
    _check(mf.grouped_matmul(x, w, off), *_reference(x, w, off), 64)
    g = _normal((3, 96), BF16, 3)
    _check(mf.grouped_matmul_backward_right(g, x, off), *_reference_right(x, g, off), 3)
    y = mf.grouped_matmul(w[0, :3, :64].contiguous(), _normal((2, 64, 64), BF16, 4), off, out=x)
    assert y is x
    _check(x, *_reference(w[0, :3, :64].contiguous(), _normal((2, 64, 64), BF16, 4), off), 64)
    stack = base.as_strided((2, 8, 8), (2 * ld, 8, 1))
    stack.copy_(_normal((2, 8, 8), BF16, 5))
    a = _normal((3, 8), BF16, 6)
    _check(mf.grouped_matmul(a, stack, off), *_reference(a, stack, off), 8)
    keep = _normal((3, 8), BF16, 7)
    mf.grouped_matmul_backward_right(keep, a, off, out=stack)
    _check(stack, *_reference_right(a, keep, off), 3)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_the_most_groups_and_many_rows(dtype):
    """1024 groups, most of them empty, and more rows than a grid dimension holds."""
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    pick = torch.randint(0, 1024, (300,), generator=g, device="cuda") // 7 * 7
    off = torch.searchsorted(pick.sort().values.contiguous(), torch.arange(1025, device="cuda")).int()
    x, w = _normal((300, 48), dtype, 1), _normal((1024, 48, 40), dtype, 2)
    _check(mf.grouped_matmul(x, w, off), *_reference(x, w, off), 48)
    d = _normal((300, 40), dtype, 3)
    _check(mf.grouped_matmul_backward_right(d, x, off), *_reference_right(x, d, off), 300)
    x, w = _normal((70001, 16), dtype, 4), _normal((2, 16, 24), dtype, 5)
    off = _offsets([65537, 4464])
    _check(mf.grouped_matmul(x, w, off), *_reference(x, w, off), 16)
    d = _normal((70001, 24), dtype, 6)
    y, s = _reference_right(x, d, off)
    got = mf.grouped_matmul_backward_right(d, x, off)
    _check(got, y, s, 70001)


@pytest.mark.parametrize("bad", [[0, 5, 3, 10], [-4, 2, 2, 6], [0, 4, 4, 99], [20, 20, 20, 20], [9, 0, 0, 0]])
def test_bad_offsets_are_clamped_and_reported(bad):
    x, g, w = _normal((10, 16), F32, 1), _normal((10, 24), F32, 2), _normal((3, 16, 24), F32, 3)
    off = torch.tensor(bad, dtype=torch.int32, device="cuda")
    fixed = [min(max(bad[0], 0), 10)]
    for v in bad[1:]:
        fixed.append(min(max(v, fixed[-1]), 10))
    fixed = torch.tensor(fixed, dtype=torch.int32, device="cuda")
    mf.device_status()
    y = mf.grouped_matmul(x, w, off)
    with pytest.raises(mf.InvalidArgumentError):
        mf.sync()
    _check(y, *_reference(x, w, fixed), 16)
    d = mf.grouped_matmul_backward_right(g, x, off)
    assert mf.device_status() != 0
    _check(d, *_reference_right(x, g, fixed), 10)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_gradients_against_differences(dtype):
    """<G, Y(X, W)> is linear in X and in W, so a central difference of step 1 is its gradient up to rounding."""
    sizes, k, n = [12, 0, 55], 48, 56
    off = _offsets(sizes)
    small = lambda shape, seed: (_normal(shape, F32, seed) * 8).round().to(dtype) / 8  # noqa: E731
    x, dx, g = small((67, k), 1), small((67, k), 2), small((67, n), 3)
    w, dw = small((3, k, n), 4), small((3, k, n), 5)
    out = lambda a, b: mf.grouped_matmul(a, b, off, out=torch.empty(67, n, device="cuda")).double()  # noqa: E731
    gl, gr = mf.grouped_matmul_backward_left(g, w, off), mf.grouped_matmul_backward_right(g, x, off)
    for up, down, grad, step, base in (((x + dx, w), (x - dx, w), gl, dx, x), ((x, w + dw), (x, w - dw), gr, dw, w)):
        difference = ((out(*up) - out(*down)) / 2 * g.double()).sum()
        product = (grad.double() * step.double()).sum()
        # rounding of the gradient to its type, and of x +- dx (w +- dw) to theirs
        half = torch.finfo(dtype).eps / 2
        tol = half * (grad.double() * step.double()).abs().sum() + 2 * half * _sum_abs(x, dx, w, dw, g, off)
        assert abs(difference - product) <= tol + 1e-5 * abs(product)


def _sum_abs(x, dx, w, dw, g, off):
    y, s = _reference(x.abs() + dx.abs(), w.abs() + dw.abs(), off)
    return (s * g.abs().double()).sum()


def test_streams_graphs_and_two_calls_at_once():
    sizes, k, n = [100, 28, 0, 200], 256, 384
    off = _offsets(sizes)
    x, g, w = _normal((328, k), BF16, 1), _normal((328, n), BF16, 2), _normal((4, k, n), BF16, 3)
    y, s = _reference(x, w, off)
    torch.cuda.synchronize()
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    got = [mf.grouped_matmul(x, w, off, stream=st) for st in (side, other) for _ in range(3)]
    with torch.cuda.stream(side):
        got.append(mf.grouped_matmul(x, w, off))
    torch.cuda.synchronize()
    for v in got:
        assert torch.equal(v, got[0])
    _check(got[0], y, s, k)
    # a captured step follows what its buffers hold at replay, offsets included
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = mf.grouped_matmul(x, w, off)
        dx = mf.grouped_matmul_backward_left(g, w, off)
        dw = mf.grouped_matmul_backward_right(g, x, off)
    for sizes in ([328, 0, 0, 0], [1, 2, 3, 4], [0, 164, 164, 0]):
        off.copy_(_offsets(sizes))
        x.copy_(_normal((328, k), BF16, sizes[0] + 5))
        graph.replay()
        _check(out, *_reference(x, w, off), k)
        _check(dx, *_reference(g, w.transpose(1, 2), off), n)
        _check(dw, *_reference_right(x, g, off), 328)


def test_results_do_not_depend_on_the_run():
    sizes = [256, 3, 0, 700, 65]
    off = _offsets(sizes)
    for dtype in (F32, BF16):
        x, g, w = _normal((1024, 1000), dtype, 1), _normal((1024, 200), dtype, 2), _normal((5, 1000, 200), dtype, 3)
        first = None
        for _ in range(5):
            got = (mf.grouped_matmul(x, w, off), mf.grouped_matmul_backward_left(g, w, off),
                   mf.grouped_matmul_backward_right(g, x, off))
            mf.sync()
            first = first or got
            assert all(torch.equal(a, b) for a, b in zip(got, first))


def test_refusals_on_device_tensors():
    x, w = _normal((4, 8), F32, 1), _normal((2, 8, 8), F32, 2)
    off = _offsets([2, 2])
    with pytest.raises(mf.InvalidArgumentError):
        mf.grouped_matmul(x, w, off, out=x)
    with pytest.raises(mf.InvalidArgumentError):
        mf.grouped_matmul(x, w, off, out=torch.empty(4, 8, device="cuda", dtype=F16))
    with pytest.raises(mf.ShapeMismatchError):
        mf.grouped_matmul(x, w, off, out=torch.empty(4, 9, device="cuda"))
    with pytest.raises(mf.InvalidArgumentError):
        mf.grouped_matmul(x, w, off.cpu())
    with pytest.raises(mf.InvalidArgumentError):
        mf.grouped_matmul_backward_right(x, x, off, out=torch.empty(1, 8, 8, device="cuda").expand(2, 8, 8))
    with pytest.raises(ValueError):
        mf.grouped_matmul(x, w, off, precision=5)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=str)
@pytest.mark.parametrize("cut", [0, 1])
@pytest.mark.parametrize("sizes", [[70, 130, 3], [20, 9]], ids=str)
def test_long_sums_of_16_bit_operands_do_not_drift(dtype, cut, sizes):
    """All products positive and FP32 outputs. Within 512 of the contraction the tensor core truncates, twice per 16:
    2 * 32 U of that chunk's sum; chunks are added with rounding, U / 2 of the sum each: U (64 + k / 1024) S in all, 80 U S
    = 9.5e-6 S at k = 16384. Truncation over the whole contraction takes 8e-5."""
    k, n, rows = 16384, 136, sum(sizes)
    off = _offsets(sizes)
    bound = lambda s: U * (64 + k / 1024) * s  # noqa: E731
    x = _normal((rows, k + 8), dtype, 1).abs()[:, cut:cut + k]
    w = _normal((len(sizes), n, k + 8), dtype, 2).abs()[:, :, cut:cut + k]
    out = torch.empty(rows, n, device="cuda")
    y, s = _reference(x, w.transpose(1, 2), off)
    assert ((mf.grouped_matmul(x, w, off, True, out=out).double() - y).abs() <= bound(s)).all()
    v = _normal((len(sizes), k, n + 8), dtype, 3).abs()[:, :, cut:cut + n]
    y, s = _reference(x, v, off)
    assert ((mf.grouped_matmul(x, v, off, out=out).double() - y).abs() <= bound(s)).all()
    a, g = _normal((k, sizes[0] + 8), dtype, 4).abs()[:, cut:cut + sizes[0]], _normal((k, 80), dtype, 5).abs()[:, cut:cut + 72]
    off = _offsets([k])
    dw = torch.empty(1, sizes[0], 72, device="cuda")
    y, s = _reference_right(a, g, off)
    assert ((mf.grouped_matmul_backward_right(g, a, off, out=dw).double() - y).abs() <= bound(s)).all()
    mf.sync()


@pytest.mark.parametrize("dtype", [F16, BF16], ids=str)
@pytest.mark.parametrize("groups,most,k,n", [(64, 40, 512, 1000), (512, 40, 72, 128), (256, 250, 128, 640), (64, 250, 512, 640)])
def test_weight_gradient_of_many_ragged_groups(dtype, groups, most, k, n):
    """Six and more tiles per SM pair, nearly all of them ending inside a 16-row step and one or two stages long, so that
    cleared rows of consecutive tiles are handed over in quick succession; for n = 128 and 640 the second SM's half of
    some tiles lies outside the operand and is filled sooner than the first's."""
    g = torch.Generator()
    g.manual_seed(groups + most)
    off = _offsets(torch.randint(0, most // 2, (groups,), generator=g).mul(2).add(1).tolist())
    rows = int(off[-1])
    x, d = _normal((rows, k), dtype, 1), _normal((rows, n), dtype, 2)
    mf.device_status()
    first = mf.grouped_matmul_backward_right(d, x, off)
    _check(first, *_reference_right(x, d, off), most)
    for _ in range(10):
        assert torch.equal(mf.grouped_matmul_backward_right(d, x, off), first)
    assert mf.device_status() == 0


def test_bad_offsets_are_no_other_calls_error():
    """Calls that wait for work of their own neither fail by them nor take the report away from sync()."""
    from matrixflash_pro_b200.distributed import sgemm_multi
    x, w = _normal((10, 16), F32, 1), _normal((1, 16, 24), F32, 2)
    a = _normal((128, 128), F32, 3)
    plan = mf.GemmPlan(128, 128, 128, mf.GemmOptions())
    calls = [lambda: plan.tune(a, a, torch.empty_like(a)), lambda: mf.probe_tf32_mma_tflops(), lambda: mf.cuda_sync(0),
             lambda: sgemm_multi([a], a, [torch.empty_like(a)])]
    for call in calls:
        mf.device_status()
        mf.grouped_matmul(x, w, torch.tensor([0, 11], dtype=torch.int32, device="cuda"))
        torch.cuda.synchronize()
        call()
        with pytest.raises(mf.InvalidArgumentError):
            mf.sync()
        mf.sync()


@pytest.mark.parametrize("e", [-110, -118, -126, -136])
def test_values_below_the_third_terms_range(e):
    """Under 2^-110 a value's third BF16 term falls below that type's smallest number, 2^-133: each loses up to 2^-134
    more than elsewhere."""
    x = torch.ldexp(_normal((70, 200), F32, 1).double(), torch.tensor(e, device="cuda")).float()
    w = _normal((1, 200, 96), F32, 2)
    off = _offsets([70])
    y, s = _reference(x, w, off)
    got = mf.grouped_matmul(x, w, off)
    mf.sync()
    assert ((got.double() - y).abs() <= _bound(y, s, 200, F32) + 2.0 ** -134 * w[0].double().abs().sum(0)).all()
