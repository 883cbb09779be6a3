"""Operators of mixture-of-experts layers: what is measured.

Three families, as one model uses them in turn. ``grouped_matmul`` and its two gradients multiply rows that
are sorted by expert with the experts' weights (training, prefill, batched decoding); ``quantize_int4`` and
``dequantize_int4`` store trained weights in 4 bits with a scale per group; ``gemv_int4`` decodes a few
tokens from those weights, dense or one expert per row.

``run`` computes the plain forms with elementary torch operations in FP32 (FP64 where a rounding to a
4-bit code could turn on the last bit), or, where ``own`` is set, makes the framework's calls.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


# ------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # One decoding step of a batch of 16 sequences, top-2 of 32 experts: one row or two an expert.
        dict(name="grouped_decode_bf16", op="grouped", type="bf16", experts=32, rows=32, spare=0, k=2048, n=1024,
             trans=False, skew=0.0),
        # Prefill or a training step's forward through the 4096 -> 11008 projection.
        dict(name="grouped_prefill_bf16", op="grouped", type="bf16", experts=8, rows=8192, spare=0, k=4096, n=11008,
             trans=False, skew=0.3),
        # The FP32 layer, weights stored [out, in], in a buffer with spare rows, some experts without rows.
        dict(name="grouped_f32", op="grouped", type="f32", experts=16, rows=3000, spare=72, k=1024, n=2048,
             trans=True, skew=1.0),
        # Input gradient, odd widths: rows of the operands start at any 2-byte address.
        dict(name="grad_left_f16_odd", op="grad_left", type="f16", experts=7, rows=1777, spare=0, k=1001, n=1531,
             trans=False, skew=0.5),
        # Input gradient of the ordinary projection.
        dict(name="grad_left_bf16", op="grad_left", type="bf16", experts=8, rows=4096, spare=0, k=2048, n=4096,
             trans=False, skew=0.3),
        # Weight gradient of the same projection.
        dict(name="grad_right_bf16", op="grad_right", type="bf16", experts=8, rows=4096, spare=0, k=2048, n=4096,
             trans=False, skew=0.3),
        # Weight gradient of many small experts in FP32, skewed, some of them empty.
        dict(name="grad_right_f32", op="grad_right", type="f32", experts=64, rows=2000, spare=48, k=512, n=1000,
             trans=False, skew=1.2),
        # One token through the 4096 -> 11008 projection.
        dict(name="int4_token_f16", op="gemv", type="f16", experts=0, rows=1, k=4096, n=11008, group=128, zeros=False),
        # A few FP32 rows through a small odd layer: latency.
        dict(name="int4_small_f32", op="gemv", type="f32", experts=0, rows=5, k=1000, n=1023, group=32, zeros=True),
        # Eight tokens, top-2 of 16 experts.
        dict(name="int4_experts_bf16", op="gemv", type="bf16", experts=16, rows=16, k=2048, n=4096, group=64,
             zeros=True),
        # Storing the projection's weights and reading them back.
        dict(name="quantize_bf16", op="quantize", type="bf16", experts=1, k=4096, n=11008, group=128, zeros=True),
        # A small odd FP32 stack, symmetric.
        dict(name="quantize_f32_odd", op="quantize", type="f32", experts=3, k=777, n=515, group=32, zeros=False),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _size(rng, low, high):
    """Half of the sizes are multiples of 64, the others whatever comes."""
    v = _spread(rng, low, high)
    return max(64, v // 64 * 64) if high >= 64 and rng.random() < 0.5 else v


def draw(rng):
    op = rng.choice(["grouped", "grouped", "grad_left", "grad_right", "gemv", "gemv", "quantize"])
    kind = rng.choice(["f32", "f16", "bf16"])
    if op in ("grouped", "grad_left", "grad_right"):
        while True:
            c = dict(op=op, type=kind, experts=_spread(rng, 1, 64), rows=_spread(rng, 1, 8192), spare=rng.choice([0, 0, 5, 64]),
                     k=_size(rng, 24, 4096), n=_size(rng, 24, 11008), trans=rng.random() < 0.4, skew=rng.choice([0.0, 0.3, 1.0]))
            if c["experts"] * c["k"] * c["n"] <= 3e8 and c["rows"] * c["k"] * c["n"] <= 1e11:
                return c
    if op == "gemv":
        while True:
            c = dict(op=op, type=kind, experts=rng.choice([0, 0, 4, 16, 64]), rows=_spread(rng, 1, 16), k=_size(rng, 32, 11008),
                     n=_size(rng, 32, 11008), group=rng.choice([32, 64, 128]), zeros=rng.random() < 0.5)
            if max(1, c["experts"]) * c["k"] * c["n"] <= 3e8 and (not c["experts"] or c["rows"] * c["k"] * c["n"] <= 4e8):
                return c
    return dict(op=op, type=kind, experts=rng.choice([1, 1, 2, 5]), k=_size(rng, 32, 4096), n=_size(rng, 32, 4096),
                group=rng.choice([32, 64, 128]), zeros=rng.random() < 0.5)


def _sizes(case):
    """Rows of each expert: fixed by the case, so that the work is; which expert has how many goes by the seed."""
    rng = random.Random("%d %d %g" % (case["experts"], case["rows"], case["skew"]))
    weights = [math.exp(case["skew"] * rng.gauss(0, 1)) for _ in range(case["experts"])]
    sizes = [0] * case["experts"]
    for e in rng.choices(range(case["experts"]), weights, k=case["rows"]):
        sizes[e] += 1
    return sizes


def _chosen(case):
    """How many rows each used expert of a decoding call gets (the work's experts), as _sizes."""
    rng = random.Random("%d %d" % (case["experts"], case["rows"]))
    return [rng.randrange(case["experts"]) for _ in range(case["rows"])]


# ------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    kind = DTYPES[case["type"]]
    k, n = case["k"], case["n"]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(kind)

    state = dict(case=case)
    if case["op"] in ("grouped", "grad_left", "grad_right"):
        experts, total = case["experts"], case["rows"] + case["spare"]
        sizes = _sizes(case)
        random.Random(seed).shuffle(sizes)
        ends = [0]
        for s in sizes:
            ends.append(ends[-1] + s)
        state["offsets"] = torch.tensor(ends, dtype=torch.int32, device="cuda")
        state["most"] = max(max(sizes), case["spare"], 1)
        if case["op"] != "grad_left":
            state["x"] = normal(total, k)
        if case["op"] != "grouped":
            state["grad"] = normal(total, n)
        if case["op"] != "grad_right":
            state["w"] = normal(experts, *((n, k) if case["trans"] else (k, n)), scale=k ** -0.5)
        return state
    group = case["group"]
    groups = -(-k // group)
    stack = (case["experts"],) if case["experts"] else ()
    if case["op"] == "gemv":
        state["packed"] = torch.randint(0, 256, (*stack, n, -(-k // 32) * 16), generator=g, device="cuda", dtype=torch.uint8)
        state["scales"] = ((torch.rand(*stack, n, groups, generator=g, device="cuda") + 0.5) * (0.2 * k ** -0.5)).to(kind)
        state["zeros"] = torch.randint(5, 11, (*stack, n, groups), generator=g, device="cuda", dtype=torch.uint8) if case["zeros"] else None
        state["x"] = normal(case["rows"], k)
        state["experts"] = None
        if stack:
            names = list(range(case["experts"]))
            random.Random(seed).shuffle(names)
            state["experts"] = torch.tensor([names[e] for e in _chosen(case)], dtype=torch.int32, device="cuda")
        return state
    state["w"] = normal(*stack, n, k, scale=k ** -0.5)
    return state


# ------------------------------------------------------------------------------------------ one pass
def run(state):
    return _own(state) if own else _plain(state)


def _own(state):
    import matrixflash_pro_b200 as mf

    case = state["case"]
    if case["op"] == "grouped":
        return mf.grouped_matmul(state["x"], state["w"], state["offsets"], transpose_right=case["trans"])
    if case["op"] == "grad_left":
        return mf.grouped_matmul_backward_left(state["grad"], state["w"], state["offsets"], transpose_right=case["trans"])
    if case["op"] == "grad_right":
        return mf.grouped_matmul_backward_right(state["grad"], state["x"], state["offsets"], transpose_right=case["trans"])
    if case["op"] == "gemv":
        if "matrix" not in state:  # the handle that a program makes when it loads its weights
            state["matrix"] = mf.Int4Matrix(state["packed"], state["scales"], state["zeros"], case["k"], case["group"])
        return mf.gemv_int4(state["matrix"], state["x"], experts=state["experts"])
    matrix = mf.quantize_int4(state["w"], case["group"], symmetric=not case["zeros"])
    return {"values": mf.dequantize_int4(matrix, state["w"].dtype), "scales": matrix.scales}


def _slots(state, total):
    """(expert, place within it) of each row; the spare rows behind the last expert go to one more."""
    offsets = state["offsets"].long()
    rows = torch.arange(total, device="cuda")
    expert = torch.searchsorted(offsets[1:].contiguous(), rows, right=True)
    return expert, rows - offsets[expert]


def _padded(t, state, expert, place):
    wide = torch.zeros(state["case"]["experts"] + 1, state["most"], t.shape[1], device="cuda")
    wide[expert, place] = t.float()
    return wide


def _codes(packed, k):
    return torch.stack((packed & 15, packed >> 4), -1).flatten(-2)[..., :k]


def _plain(state):
    case = state["case"]
    if case["op"] in ("grouped", "grad_left"):
        t = state["x"] if case["op"] == "grouped" else state["grad"]
        expert, place = _slots(state, t.shape[0])
        wide = _padded(t, state, expert, place)
        w = state["w"].float()
        if case["trans"] != (case["op"] == "grad_left"):
            w = w.transpose(1, 2)
        y = torch.zeros(wide.shape[0], wide.shape[1], w.shape[2], device="cuda")
        torch.bmm(wide[:-1], w, out=y[:-1])
        return y[expert, place].to(t.dtype)
    if case["op"] == "grad_right":
        expert, place = _slots(state, state["x"].shape[0])
        x, d = (_padded(state[name], state, expert, place)[:-1] for name in ("x", "grad"))
        left, right = (d, x) if case["trans"] else (x, d)
        return torch.bmm(left.transpose(1, 2), right).to(state["x"].dtype)
    k, group = case["k"], case["group"]
    if case["op"] == "gemv":
        scales = state["scales"].float().repeat_interleave(group, -1)[..., :k]
        zeros = 8.0 if state["zeros"] is None else state["zeros"].float().repeat_interleave(group, -1)[..., :k]
        w = (_codes(state["packed"], k).float() - zeros) * scales
        x = state["x"].float()
        if state["experts"] is None:
            return (x @ w.t()).to(state["x"].dtype)
        return torch.bmm(w[state["experts"].long()], x[:, :, None])[:, :, 0].to(state["x"].dtype)
    w = state["w"]
    groups = -(-k // group)
    wide = torch.zeros(*w.shape[:-1], groups * group, device="cuda", dtype=torch.float64)
    wide[..., :k] = w
    wide = wide.view(*w.shape[:-1], groups, group)
    if case["zeros"]:
        low, high = wide.amin(-1).clamp(max=0), wide.amax(-1).clamp(min=0)
        scales = (high - low) / 15
    else:
        scales = wide.abs().amax(-1) / 7
    scales = scales.clamp(max=torch.finfo(w.dtype).max).to(w.dtype)
    scales = torch.where(scales == 0, 1, scales)
    step = scales.double()
    zeros = torch.round(-low / step).clamp(0, 15) if case["zeros"] else torch.full_like(step, 8.0)
    codes = (torch.round(wide / step[..., None]) + zeros[..., None]).clamp(0, 15)
    values = ((codes - zeros[..., None]) * step[..., None]).flatten(-2)[..., :k].to(w.dtype)
    return {"values": values, "scales": scales}


# ------------------------------------------------------------------------------------------ the floor
def work(case):
    b, k, n = BYTES[case["type"]], case["k"], case["n"]
    if case["op"] in ("grouped", "grad_left", "grad_right"):
        used = sum(s > 0 for s in _sizes(case))
        rows, total = case["rows"], case["rows"] + case["spare"]
        if case["op"] == "grad_right":
            moved = rows * (k + n) + case["experts"] * k * n
        else:
            wide, out = (k, n) if case["op"] == "grouped" else (n, k)
            moved = rows * wide + used * k * n + total * out
        return {"bytes": moved * b, "flops": 2 * rows * k * n}
    groups = -(-k // case["group"])
    weights = n * (-(-k // 2) + groups * (b + (1 if case["zeros"] else 0)))
    if case["op"] == "gemv":
        used = len(set(_chosen(case))) if case["experts"] else 1
        return {"bytes": used * weights + case["rows"] * (k + n) * b, "flops": 2 * case["rows"] * k * n}
    # weights read, codes written; codes read back, values written
    return {"bytes": case["experts"] * (2 * n * k * b + 2 * weights), "flops": 6 * case["experts"] * n * k}


# ------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    k, n = case["k"], case["n"]
    if case["op"] in ("grouped", "grad_left", "grad_right"):
        ends = state["offsets"].tolist()
        spans = [(e, slice(ends[e], ends[e + 1])) for e in range(case["experts"]) if ends[e + 1] > ends[e]]
        if case["op"] == "grad_right":
            y = torch.zeros(case["experts"], *((n, k) if case["trans"] else (k, n)), device="cuda", dtype=torch.float64)
            for e, s in spans:
                x, d = state["x"][s].double(), state["grad"][s].double()
                y[e] = d.mT @ x if case["trans"] else x.mT @ d
            return y
        t, wide = (state["x"], n) if case["op"] == "grouped" else (state["grad"], k)
        y = torch.zeros(t.shape[0], wide, device="cuda", dtype=torch.float64)
        for e, s in spans:
            w = state["w"][e].double()
            w = w.mT if case["trans"] else w  # now [k, n]
            y[s] = t[s].double() @ (w if case["op"] == "grouped" else w.mT)
        return y
    group = case["group"]
    at = torch.arange(k, device="cuda")
    if case["op"] == "gemv":
        rows = []
        for r in range(case["rows"]):
            pick = (lambda t: t) if state["experts"] is None else (lambda t, e=int(state["experts"][r]): t[e])
            code = (pick(state["packed"])[:, at // 2].int() >> (4 * (at % 2)).int()) % 16
            zero = 8 if state["zeros"] is None else pick(state["zeros"])[:, at // group].int()
            w = (code - zero).double() * pick(state["scales"])[:, at // group].double()
            rows.append(w @ state["x"][r].double())
        return torch.stack(rows)
    w = state["w"]
    values, scales = torch.empty(w.shape, device="cuda", dtype=torch.float64), []
    for first in range(0, k, group):
        v = w[..., first:first + group].double()
        if case["zeros"]:
            low = torch.minimum(v.min(-1).values, torch.zeros((), device="cuda", dtype=torch.float64))
            step = (torch.maximum(v.max(-1).values, torch.zeros_like(low)) - low) / 15
        else:
            step = v.abs().max(-1).values / 7
        step = step.to(w.dtype).double()  # the definition rounds the scale before anything uses it
        step[step == 0] = 1.0
        zero = torch.round(-low / step) if case["zeros"] else torch.full_like(step, 8.0)
        code = torch.round(v / step[..., None]) + zero[..., None]
        code = torch.minimum(torch.maximum(code, torch.zeros_like(code)), torch.full_like(code, 15.0))
        values[..., first:first + group] = (code - zero[..., None]) * step[..., None]
        scales.append(step)
    return {"values": values, "scales": torch.stack(scales, -1)}
