"""GPU tier: the expert operators together, as a mixture-of-experts layer uses them.

Rows are routed to experts and sorted, pass two grouped products (a training step takes their gradients), the
trained weights are stored in 4 bits, and single tokens are decoded from those."""
import pytest
import torch

import matrixflash_pro_b200 as mf

pytestmark = pytest.mark.gpu


def _route(tokens, experts, top, seed):
    """(order, offsets, expert ids in the tokens' order): `top` different experts a token, rows sorted by expert."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    ids = torch.rand(tokens, experts, generator=g, device="cuda").topk(top, -1).indices.flatten()
    order = torch.argsort(ids, stable=True)
    ends = torch.searchsorted(ids[order].contiguous(), torch.arange(experts, device="cuda"), right=True)
    return order, torch.cat([ends.new_zeros(1), ends]).int(), ids


class _Layer(torch.autograd.Function):
    """Y = relu(X W1) W2 by expert; how a user ties the three products to autograd."""

    @staticmethod
    def forward(ctx, x, w1, w2, off):
        h = mf.grouped_matmul(x, w1, off).relu_()
        ctx.save_for_backward(x, w1, w2, off, h)
        return mf.grouped_matmul(h, w2, off)

    @staticmethod
    def backward(ctx, grad):
        x, w1, w2, off, h = ctx.saved_tensors
        grad = grad.contiguous()
        dh = mf.grouped_matmul_backward_left(grad, w2, off) * (h > 0)
        return (mf.grouped_matmul_backward_left(dh, w1, off), mf.grouped_matmul_backward_right(dh, x, off),
                mf.grouped_matmul_backward_right(grad, h, off), None)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_train_store_decode(dtype):
    tokens, experts, top, d, f = 60, 6, 2, 96, 160
    order, off, ids = _route(tokens, experts, top, 1)
    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    x = torch.randn(tokens, d, generator=g, device="cuda").to(dtype)
    w1 = (torch.randn(experts, d, f, generator=g, device="cuda") * d ** -0.5).to(dtype).requires_grad_()
    w2 = (torch.randn(experts, f, d, generator=g, device="cuda") * f ** -0.5).to(dtype).requires_grad_()
    rows = x[order // top].requires_grad_()
    y = _Layer.apply(rows, w1, w2, off)
    up = torch.randn(y.shape, generator=g, device="cuda").to(dtype)
    y.backward(up)
    mf.sync()
    # the same step in FP64, expert by expert
    ref = [t.detach().double().requires_grad_() for t in (rows, w1, w2)]
    o = off.tolist()
    parts = [(ref[0][o[e]:o[e + 1]] @ ref[1][e]).relu() @ ref[2][e] for e in range(experts)]
    y64 = torch.cat(parts)
    y64.backward(up.double())
    # rounding of the hidden rows and of the result: a few half steps of the type, normwise
    tol = 4 * torch.finfo(dtype).eps
    for got, want in [(y, y64)] + [(a.grad, b.grad) for a, b in zip((rows, w1, w2), ref)]:
        assert ((got.double() - want).norm() / want.norm()).item() <= tol

    # decoding: the weights in 4 bits, a row per token and chosen expert, against the products of what is stored
    q1 = mf.quantize_int4(w1.detach().transpose(1, 2).contiguous(), 32)
    q2 = mf.quantize_int4(w2.detach().transpose(1, 2).contiguous(), 64, symmetric=True)
    ids8 = ids[:8 * top].int()
    row8 = x[:8].repeat_interleave(top, 0)
    h = mf.gemv_int4(q1, row8, experts=ids8).relu_()
    out = mf.gemv_int4(q2, h, experts=ids8)
    sort8 = torch.argsort(ids8, stable=True)
    ends = torch.searchsorted(ids8[sort8].contiguous(), torch.arange(experts, device="cuda", dtype=torch.int32), right=True)
    off8 = torch.cat([ends.new_zeros(1), ends]).int()
    d1, d2 = mf.dequantize_int4(q1, torch.float32), mf.dequantize_int4(q2, torch.float32)
    h2 = mf.grouped_matmul(row8[sort8].float(), d1, off8, transpose_right=True).relu_().to(dtype)
    out2 = mf.grouped_matmul(h2.float(), d2, off8, transpose_right=True)
    mf.sync()
    assert ((out[sort8].double() - out2.double()).norm() / out2.double().norm()).item() <= tol
    # and the step from the trained weights to 4 bits is a rounding to within half a step of each group's scale
    step = q1.scales.float().repeat_interleave(32, -1)[..., :d]
    exact = (d1 - w1.detach().transpose(1, 2).float()).abs()
    # a clamped end of the range adds the rounding of the scale (its half step, 15 codes) and of the zero point
    assert (exact <= step * (1.0 + 15 * torch.finfo(dtype).eps / 2)).all()


_FIRST_CALLS = """
import torch, matrixflash_pro_b200 as mf
x = torch.randn(40, 64, device="cuda").bfloat16()
w = torch.randn(3, 64, 96, device="cuda").bfloat16()
g = torch.randn(40, 96, device="cuda").bfloat16()
off = torch.tensor([0, 10, 10, 40], dtype=torch.int32, device="cuda")
ids = torch.tensor([0, 2], dtype=torch.int32, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = mf.grouped_matmul(x, w, off)
    d = mf.grouped_matmul_backward_right(g, x, off)
    q = mf.quantize_int4(w.transpose(1, 2).contiguous(), 32)
    z = mf.gemv_int4(q, x[:2], experts=ids)
    b = mf.dequantize_int4(q)
graph.replay()
mf.sync()
ref = torch.cat([x[:10].double() @ w[0].double(), x[10:].double() @ w[2].double()])
assert ((y.double() - ref).norm() / ref.norm()).item() < 4e-3
ref = torch.stack([b[0].double() @ x[0].double(), b[2].double() @ x[1].double()])
assert ((z.double() - ref).norm() / ref.norm()).item() < 8e-3
print("captured")
"""


def test_the_first_calls_of_a_process_can_be_captured():
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    env = dict(os.environ, PYTHONPATH=root)
    r = subprocess.run([sys.executable, "-c", _FIRST_CALLS], cwd=root, env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]
