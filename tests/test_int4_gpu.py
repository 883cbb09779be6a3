"""GPU tier: 4-bit weights against their definition in FP64.

Codes, zero points and scales are equal to the definition's, and so is what is read back (one rounding of an
exact value). gemv_int4, elementwise: |y - y64| <= 2^-23 (k / 8 + 32) S + r |y64| as for the grouped products, S =
sum |w_j x_j|, r half a step of a 16-bit output (FP32 rows enter as three BF16 terms, which hold them exactly)."""
import pytest
import torch

import matrixflash_pro_b200 as mf

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = 2.0 ** -23


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(shape, dtype, seed, scale=1.0):
    return (torch.randn(shape, generator=_gen(seed), device="cuda") * scale).to(dtype)


def _unpack(packed, k):
    return torch.stack((packed & 15, packed >> 4), -1).flatten(-2)[..., :k].long()


def _spread(t, group, k):
    return t.repeat_interleave(group, -1)[..., :k]


def _values(m):
    """FP64 weights of a matrix."""
    z = 8 if m.zeros is None else _spread(m.zeros.long(), m.group, m.k)
    return (_unpack(m.packed, m.k) - z).double() * _spread(m.scales.double(), m.group, m.k)


def _quantised(w, group, symmetric, scale_dtype):
    """(codes, scales, zeros) by the definition: FP64, the scale rounded (through FP32) before it is used."""
    k = w.shape[-1]
    groups = -(-k // group)
    wide = torch.zeros(*w.shape[:-1], groups * group, dtype=torch.float64, device="cuda")
    wide[..., :k] = w
    wide = wide.unflatten(-1, (groups, group))
    if symmetric:
        s = wide.abs().amax(-1) / 7
    else:
        lo, hi = wide.amin(-1).clamp(max=0), wide.amax(-1).clamp(min=0)
        s = (hi - lo) / 15
    s = s.clamp(max=torch.finfo(scale_dtype).max).to(scale_dtype)
    s = torch.where(s == 0, torch.ones_like(s), s)
    step = s.double()
    z = torch.full_like(step, 8) if symmetric else torch.round(-lo / step).clamp(0, 15)
    q = (torch.round(wide / step[..., None]) + z[..., None]).clamp(0, 15)
    return q.flatten(-2)[..., :k].long(), s, z.long()


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("symmetric", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantise_and_read_back(dtype, symmetric, group):
    for i, shape in enumerate([(1, 1), (3, 31), (5, 32), (16, 128), (7, 129), (2, 9, 500), (4, 1, 1024), (33, 4097)]):
        w = _normal(shape, dtype, i, 0.05)
        for scale_dtype in ((None, F32, F16, BF16) if i in (4, 5) else (None,)):
            m = mf.quantize_int4(w, group, symmetric, scale_dtype)
            q, s, z = _quantised(w, group, symmetric, scale_dtype or dtype)
            mf.sync()
            assert m.shape == w.shape and m.scales.dtype == (scale_dtype or dtype)
            assert torch.equal(m.scales, s)
            assert (m.zeros is None) == symmetric and (symmetric or torch.equal(m.zeros.long(), z))
            assert torch.equal(_unpack(m.packed, w.shape[-1]), q)
            for out in (None, F32, F16, BF16):
                got = mf.dequantize_int4(m, out)
                assert torch.equal(got, _values(m).float().to(out or m.scales.dtype))


@pytest.mark.parametrize("symmetric", [False, True])
def test_quantise_on_the_borders(symmetric):
    """Weights halfway between codes, groups of one value, zeros, and scales beyond the scale type's range."""
    steps = torch.arange(-15, 16, device="cuda") / 2
    rows = [torch.cat([steps * s, steps.new_full((1,), 7.5 * s)]) for s in (1.0, 0.5, 3.0, 1e-3, 0.1)]
    rows += [torch.zeros(32, device="cuda"), torch.full((32,), 2.5, device="cuda"), torch.full((32,), -2.5, device="cuda")]
    near = (steps + 0.5) * 0.7
    rows += [torch.cat([torch.nextafter(near, near.new_full((), sign * 99.0)), near.new_full((1,), 5.0)])
             for sign in (-1, 1)]
    w = torch.stack(rows)
    for dtype in (F32, F16, BF16):
        m = mf.quantize_int4(w.to(dtype), 32, symmetric)
        q, s, z = _quantised(w.to(dtype), 32, symmetric, dtype)
        mf.sync()
        assert torch.equal(m.scales, s) and torch.equal(_unpack(m.packed, 32), q)
        assert symmetric or torch.equal(m.zeros.long(), z)
    big = torch.tensor([[1e6, -3e5, 12.0, 0.0] * 8, [3e38, -3e38, 1e38, 0.0] * 8, [1e-30, -1e-31, 0.0, 0.0] * 8],
                       device="cuda")
    for scale_dtype in (F32, F16, BF16):
        m = mf.quantize_int4(big, 32, symmetric, scale_dtype)
        q, s, z = _quantised(big, 32, symmetric, scale_dtype)
        mf.sync()
        assert torch.equal(m.scales, s) and torch.equal(_unpack(m.packed, 32), q)
        assert torch.isfinite(mf.dequantize_int4(m, F32)).all()


@pytest.mark.parametrize("symmetric", [False, True])
def test_quantise_the_smallest_scales(symmetric):
    """Weights near the end of FP32's range, where a scale has no reciprocal."""
    w = _normal((40, 64), F32, 1) * torch.logspace(-44, -36, 40, device="cuda", dtype=torch.float64)[:, None]
    w = w.to(F32)
    m = mf.quantize_int4(w, 32, symmetric)
    q, s, z = _quantised(w, 32, symmetric, F32)
    mf.sync()
    assert torch.equal(m.scales, s) and torch.equal(_unpack(m.packed, 64), q)
    assert symmetric or torch.equal(m.zeros.long(), z)


def test_quantise_strided_weights():
    whole = _normal((6, 40, 300), BF16, 1)
    for w in (whole[::2, 1:, 3:260], whole[:, ::3, :299], whole[1, :, 7:200], whole[:, :1, :64]):
        m = mf.quantize_int4(w, 64)
        q, s, z = _quantised(w, 64, False, BF16)
        mf.sync()
        assert torch.equal(_unpack(m.packed, w.shape[-1]), q) and torch.equal(m.scales, s)
        out = torch.full((*w.shape[:-1], w.shape[-1] + 5), 9.0, device="cuda")
        cut = out[..., 2:2 + w.shape[-1]]
        assert mf.dequantize_int4(m, out=cut) is cut
        assert torch.equal(cut, _values(m).float()) and (out[..., :2] == 9).all() and (out[..., -3:] == 9).all()


def _matrix(stack, n, k, group, zeros, dtype, seed):
    g = _gen(seed)
    lead = (stack,) if stack else ()
    groups = -(-k // group)
    packed = torch.randint(0, 256, (*lead, n, 16 * (-(-k // 32))), generator=g, device="cuda", dtype=torch.uint8)
    scales = ((torch.rand(*lead, n, groups, generator=g, device="cuda") + 0.5) * 0.1).to(dtype)
    z = torch.randint(0, 16, (*lead, n, groups), generator=g, device="cuda", dtype=torch.uint8) if zeros else None
    return mf.Int4Matrix(packed, scales, z, k, group)


def _check_gemv(y, m, x, ids=None):
    w = _values(m)
    w = w if ids is not None else w.expand(x.shape[0], *w.shape) if w.dim() == 2 else w
    for r in range(x.shape[0]):
        if ids is not None and not 0 <= ids[r] < m.experts:
            assert not y[r].any()
            continue
        wr = w[ids[r]] if ids is not None else w[r]
        ref, s = wr @ x[r].double(), wr.abs() @ x[r].double().abs()
        half = 0.0 if x.dtype == F32 else torch.finfo(x.dtype).eps / 2
        low = 0.0 if x.dtype == F32 else torch.finfo(x.dtype).smallest_normal * half
        assert ((y[r].double() - ref).abs() <= U * (m.k / 8 + 32) * s + half * ref.abs() + low).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zeros", [False, True])
def test_gemv(dtype, group, zeros):
    for i, (rows, n, k) in enumerate([(1, 1, 1), (1, 16, 32), (2, 17, 33), (3, 100, 127), (8, 64, 256), (9, 31, 1000),
                                      (16, 48, 4096), (1, 1023, 777), (5, 33, 11008), (17, 40, 512), (64, 70, 96),
                                      (1, 4096, 128), (33, 19, 1500)]):
        for scale_dtype in ((F32, F16, BF16) if i in (4, 5) else (dtype,)):
            m = _matrix(0, n, k, group, zeros, scale_dtype, i)
            x = _normal((rows, k), dtype, 50 + i)
            y = mf.gemv_int4(m, x)
            mf.sync()
            assert y.shape == (rows, n) and y.dtype == dtype
            _check_gemv(y, m, x)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=str)
@pytest.mark.parametrize("group", [32, 64, 128])
def test_gemv_by_expert(dtype, group):
    for i, (stack, n, k, ids) in enumerate([
            (4, 33, 200, [2]), (4, 33, 200, [3, 3, 0, 1, 3]), (1, 16, 64, [0] * 20), (64, 20, 96, list(range(63, -1, -1))),
            (8, 130, 1024, [7, 0, 7, 7, 2, 7, 7, 7, 7, 7, 7, 7]), (3, 48, 320, [-1, 2, -7, 0]), (5, 64, 128, [-1, -1])]):
        m = _matrix(stack, n, k, group, i % 2 == 0, dtype, i)
        x = _normal((len(ids), k), dtype, 60 + i)
        for r, e in enumerate(ids):
            if e < 0:
                x[r] = float("nan")  # a padded row: nothing of it is used
        y = mf.gemv_int4(m, x, experts=torch.tensor(ids, dtype=torch.int32, device="cuda"))
        mf.sync()
        _check_gemv(y, m, x, ids)


def test_expert_past_the_stack_is_reported():
    m = _matrix(3, 20, 64, 32, False, F16, 1)
    x = _normal((4, 64), F16, 2)
    mf.device_status()
    y = mf.gemv_int4(m, x, experts=torch.tensor([1, 3, 2, 1 << 30], dtype=torch.int32, device="cuda"))
    with pytest.raises(mf.InvalidArgumentError):
        mf.sync()
    _check_gemv(y, m, x, [1, 3, 2, 1 << 30])


def test_codes_behind_the_last_column_are_ignored():
    m = _matrix(0, 24, 45, 32, True, F32, 1)
    x = _normal((3, 45), F32, 2)
    first = mf.gemv_int4(m, x).clone()
    m.packed[:, 23:] ^= 0x5a
    m.packed[:, 22] ^= 0xf0
    assert torch.equal(mf.gemv_int4(m, x), first)
    mf.sync()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
def test_gemv_strides(dtype):
    m = _matrix(0, 75, 333, 64, True, BF16, 1)
    wide = _normal((9, 400), dtype, 2)
    for cut in (0, 1, 5):
        x = wide[:, cut:cut + 333]
        out = torch.full((9, 90), 4.0, dtype=dtype, device="cuda")
        y = out[:, cut:cut + 75]
        assert mf.gemv_int4(m, x, out=y) is y
        mf.sync()
        _check_gemv(y, m, x)
        assert (out[:, :cut] == 4).all() and (out[:, cut + 75:] == 4).all()
    x = wide[:1, :333].expand(4, 333)  # one row for all
    _check_gemv(mf.gemv_int4(m, x), m, x)


def test_non_finite_rows_stay_alone():
    m = _matrix(0, 40, 256, 128, True, F16, 1)
    for dtype in (F32, F16, BF16):
        x = _normal((6, 256), dtype, 2)
        clean = mf.gemv_int4(m, x)
        x[1, 5], x[4, 9] = float("nan"), float("inf")
        y = mf.gemv_int4(m, x)
        mf.sync()
        keep = torch.tensor([0, 2, 3, 5], device="cuda")
        assert torch.equal(y[keep], clean[keep]) and y[1].isnan().all()


def test_positions_past_32_bits():
    """A stack whose last matrix lies past 2^32 codes and 2^31 bytes."""
    n, k, stack = 8192, 8192, 66
    packed = torch.empty(stack, n, k // 2, dtype=torch.uint8, device="cuda")
    packed[-1].random_(0, 256, generator=_gen(1))
    scales = torch.full((stack, n, k // 128), 0.01, dtype=F16, device="cuda")
    m = mf.Int4Matrix(packed, scales, None, k, 128)
    x = _normal((2, k), F16, 2)
    ids = torch.tensor([stack - 1, stack - 1], dtype=torch.int32, device="cuda")
    y = mf.gemv_int4(m, x, experts=ids)
    mf.sync()
    last = mf.Int4Matrix(packed[-1], scales[-1], None, k, 128)
    _check_gemv(y, last, x)
    w = torch.empty(stack * n * k + 64, dtype=F16, device="cuda")[:stack * n * k].view(stack, n, k)
    mf.dequantize_int4(m, out=w)
    assert torch.equal(w[-1], _values(last).float().half())
    w[-1].normal_(generator=_gen(3))
    q = mf.quantize_int4(w[stack - 2:], 128)
    assert torch.equal(_unpack(q.packed[-1], k), _quantised(w[-1], 128, False, F16)[0])


def test_streams_graphs_and_two_calls_at_once():
    m = _matrix(4, 200, 640, 64, True, BF16, 1)
    x = _normal((10, 640), BF16, 2)
    ids = torch.tensor([0, 1, 2, 3, 3, 3, 0, -1, 2, 1], dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [mf.gemv_int4(m, x, experts=ids, stream=s) for s in streams for _ in range(4)]
    torch.cuda.synchronize()
    assert all(torch.equal(g, got[0]) for g in got)
    w = _normal((4, 200, 640), BF16, 3)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = mf.quantize_int4(w, 64)
        back = mf.dequantize_int4(q)
        y = mf.gemv_int4(q, x, experts=ids)
    for seed in (4, 5):
        w.copy_(_normal((4, 200, 640), BF16, seed))
        ids.copy_(torch.randint(-1, 4, (10,), generator=_gen(seed), device="cuda", dtype=torch.int32))
        graph.replay()
        mf.sync()
        assert torch.equal(_unpack(q.packed, 640), _quantised(w, 64, False, BF16)[0])
        assert torch.equal(back, _values(q).float().to(BF16))
        _check_gemv(y, q, x, ids.tolist())


def test_refusals_on_device_tensors():
    m = _matrix(0, 8, 64, 32, False, F16, 1)
    stack = _matrix(2, 8, 64, 32, False, F16, 1)
    x = _normal((3, 64), F16, 2)
    ids = torch.zeros(3, dtype=torch.int32, device="cuda")
    invalid = [lambda: mf.gemv_int4(m, x.double()), lambda: mf.gemv_int4(m, x.cpu()), lambda: mf.gemv_int4(stack, x),
               lambda: mf.gemv_int4(m, _normal((65, 64), F16, 1)), lambda: mf.gemv_int4(stack, x, experts=ids.long()),
               lambda: mf.gemv_int4(m, _normal((64, 3), F16, 1).t()), lambda: mf.gemv_int4(stack, x, experts=ids.cpu()),
               lambda: mf.gemv_int4(m, x, out=torch.empty(3, 8, device="cuda")),
               lambda: mf.gemv_int4(m, x, out=torch.empty(1, 8, device="cuda", dtype=F16).expand(3, 8)),
               lambda: mf.gemv_int4(m, x, out=x[:, :8]), lambda: mf.dequantize_int4(m, torch.float64),
               lambda: mf.Int4Matrix(m.packed[:, ::2], m.scales[:, :1].contiguous(), None, 32, 32),
               lambda: mf.Int4Matrix(m.packed.flatten()[8:136].view(8, 16), m.scales[:, :1].contiguous(), None, 32, 32),
               lambda: mf.quantize_int4(_normal((64, 8), F16, 1).t())]
    for call in invalid:
        with pytest.raises(mf.InvalidArgumentError):
            call()
    for call in (lambda: mf.gemv_int4(m, x[:, :32]), lambda: mf.gemv_int4(stack, x, experts=ids[:2]),
                 lambda: mf.gemv_int4(m, x, out=torch.empty(3, 9, device="cuda", dtype=F16)),
                 lambda: mf.dequantize_int4(m, out=torch.empty(8, 65, device="cuda"))):
        with pytest.raises(mf.ShapeMismatchError):
            call()


def test_empty_calls():
    m = _matrix(0, 8, 64, 32, False, F16, 1)
    assert mf.gemv_int4(m, torch.empty(0, 64, device="cuda", dtype=F16)).shape == (0, 8)
    none = mf.Int4Matrix(m.packed[:, :0].contiguous(), m.scales[:, :0].contiguous(), None, 0, 32)
    y = mf.gemv_int4(none, torch.empty(3, 0, device="cuda"))
    mf.sync()
    assert y.shape == (3, 8) and not y.any()
    q = mf.quantize_int4(torch.empty(0, 40, device="cuda"), 32)
    assert mf.dequantize_int4(q).shape == (0, 40)


def test_empty_stack_gives_zero_rows():
    for dtype in (F32, F16):
        q = mf.quantize_int4(torch.empty(0, 24, 64, dtype=dtype, device="cuda"), 32)
        x = _normal((3, 64), dtype, 1)
        y = mf.gemv_int4(q, x, experts=torch.full((3,), -1, dtype=torch.int32, device="cuda"))
        mf.sync()
        assert q.shape == (0, 24, 64) and y.shape == (3, 24) and not y.any()
        y = mf.gemv_int4(q, x, experts=torch.tensor([-1, 0, 5], dtype=torch.int32, device="cuda"))
        with pytest.raises(mf.InvalidArgumentError):
            mf.sync()
        assert not y.any() and mf.dequantize_int4(q).shape == (0, 24, 64)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=str)
def test_infinite_rows(dtype):
    """An infinite value gives what the products of the formula give: an infinity of the weight's sign, or NaN where the
    weight is 0 or infinities of both signs meet. The largest finite value is no infinity."""
    m = _matrix(0, 70, 300, 64, True, F32, 3)
    x = _normal((5, 300), dtype, 4)
    x[0, 7], x[1, 299], x[2, 3], x[2, 130], x[3, 64] = float("inf"), float("-inf"), float("inf"), float("inf"), torch.finfo(dtype).max
    y = mf.gemv_int4(m, x)
    mf.sync()
    ref = (x.double() @ _values(m).t())[:3]
    assert (ref == float("inf")).any() and (ref == float("-inf")).any() and ref.isnan().any()
    assert torch.equal(y[:3].double().nan_to_num(7.0, float("inf"), float("-inf")), ref.nan_to_num(7.0, float("inf"), float("-inf")))
    assert not y[3:].isnan().any() and y[4].isfinite().all()


@pytest.mark.parametrize("e", [-110, -118, -126, -136])
def test_values_below_the_third_terms_range(e):
    """Under 2^-110 a value's third BF16 term falls below that type's smallest number, 2^-133: each loses up to 2^-134
    more than elsewhere."""
    m = _matrix(0, 96, 200, 128, True, F32, 1)
    x = torch.ldexp(_normal((8, 200), F32, 2).double(), torch.tensor(e, device="cuda")).float()
    y = mf.gemv_int4(m, x)
    mf.sync()
    w = _values(m)
    ref, s = x.double() @ w.t(), x.double().abs() @ w.abs().t()
    assert ((y.double() - ref).abs() <= U * (200 / 8 + 32) * s + 2.0 ** -134 * w.abs().sum(1)).all()
