"""Measured passes of the expert-layer operators: block-scaled 8-bit products and products grouped by expert.

Four families, as an MLP layer made of experts uses them next to the dense
GEMM+SwiGLU of this library:

  quantize   rows (1 x 128 blocks) or weights (128 x 128 blocks) to e4m3 with
             one fp32 scale a block;
  fp8        x . W^T of such operands, plain or packed gate/up with SwiGLU;
  grouped    rows sorted by expert times that expert's weight, in bf16 or in
             block-scaled e4m3, plain or SwiGLU;
  backward   both gradients of the plain bf16 grouped product.

``run`` computes them in elementary torch operations in 32 bits where ``own`` is
false, and calls the library where it is true.
"""

import math
import random
import sys

import numpy as np
import torch

own = False

BLOCK = 128
E4M3_MAX = 448.0
# Blocks whose largest magnitude is below this (all-zero blocks among them)
# take it as their largest, so that 448 / amax stays finite.
AMAX_FLOOR = 2.0 ** -100
F8 = torch.float8_e4m3fn
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def _library():
    if "cuda-operator-lab_b200" not in sys.path:
        sys.path.insert(0, "cuda-operator-lab_b200")
    from cuda_operator_lab import fp8, grouped

    return fp8, grouped


# ------------------------------------------------------------------ cases


def listed():
    return [
        # one token's activations on their way into an 8-bit projection: latency
        {"name": "quantize one token", "op": "quantize", "dtype": "bf16", "m": 1, "k": 4096,
         "experts": 0},
        # a prompt's activations: memory traffic
        {"name": "quantize prompt", "op": "quantize", "dtype": "bf16", "m": 16384, "k": 4096,
         "experts": 0},
        # weights of a few experts when a checkpoint is loaded, odd height
        {"name": "quantize expert weights", "op": "quantize", "dtype": "fp32", "m": 1900,
         "k": 2064, "experts": 6},
        # one token through a square projection: reading the weight, latency
        {"name": "fp8 one token", "op": "fp8", "m": 1, "n": 4096, "k": 4096, "swiglu": False},
        # a small batch with odd sizes, the last block of k partial
        {"name": "fp8 odd batch", "op": "fp8", "m": 333, "n": 5001, "k": 2064, "swiglu": False},
        # gate/up of a long prompt, the dense MLP's widths
        {"name": "fp8 swiglu prompt", "op": "fp8", "m": 8192, "n": 14336, "k": 4096,
         "swiglu": True},
        # decoding: a few rows an expert, some experts without any
        {"name": "grouped fp8 decode", "op": "grouped", "dtype": "fp8", "t": 256, "experts": 64,
         "n": 1024, "k": 4096, "swiglu": True, "skew": 0.7, "routing": 11},
        # a prompt over experts of different popularity
        {"name": "grouped fp8 prompt", "op": "grouped", "dtype": "fp8", "t": 16384, "experts": 16,
         "n": 4096, "k": 2048, "swiglu": False, "skew": 0.5, "routing": 12},
        # a handful of rows over experts of odd width
        {"name": "grouped bf16 few rows", "op": "grouped", "dtype": "bf16", "t": 37,
         "experts": 24, "n": 1511, "k": 1000, "swiglu": False, "skew": 1.0, "routing": 13},
        # gate/up of a training or prompt batch
        {"name": "grouped bf16 swiglu", "op": "grouped", "dtype": "bf16", "t": 16384, "experts": 8,
         "n": 4096, "k": 4096, "swiglu": True, "skew": 0.5, "routing": 14},
        # a small ragged training batch, several experts without rows
        {"name": "backward ragged", "op": "backward", "t": 1100, "experts": 20, "n": 776,
         "k": 520, "skew": 1.5, "routing": 15},
        # a full training batch
        {"name": "backward batch", "op": "backward", "t": 16384, "experts": 8, "n": 2048,
         "k": 4096, "skew": 0.5, "routing": 16},
    ]


def _log_int(rng, lo, hi, multiple=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(multiple, int(round(v / multiple)) * multiple)


def draw(rng):
    flops_most = 2.0 * 8192 * 4096 * 2 * 14336
    op = rng.choice(["quantize", "fp8", "grouped", "grouped", "backward"])
    while True:
        if op == "quantize":
            weight = rng.random() < 0.4
            case = {"op": op, "dtype": rng.choice(["bf16", "fp32"]),
                    "m": _log_int(rng, 1, 16384), "k": _log_int(rng, 128, 8192, 16),
                    "experts": _log_int(rng, 1, 16) if weight else 0}
            if case["m"] * case["k"] * max(1, case["experts"]) <= 16384 * 4096:
                return case
            continue
        experts = 1 if op == "fp8" else _log_int(rng, 2, 96)
        swiglu = op != "backward" and rng.random() < 0.4
        fp8 = op == "fp8" or (op == "grouped" and rng.random() < 0.5)
        n = _log_int(rng, 128, 8192, 128 if fp8 and swiglu else 8 if op == "backward" else 1)
        k = _log_int(rng, 128, 8192, 16 if fp8 else 8)
        rows = _log_int(rng, 1, 16384)
        columns = 2 * n if swiglu else n
        flops = 2.0 * rows * columns * k * (2 if op == "backward" else 1)
        # a plain pass pads every expert to the longest one
        if flops * (4 if experts > 1 else 1) > flops_most or experts * columns * k > 6e8:
            continue
        if op == "fp8":
            return {"op": op, "m": rows, "n": n, "k": k, "swiglu": swiglu}
        case = {"op": op, "t": rows, "experts": experts, "n": n, "k": k,
                "skew": round(rng.uniform(0.2, 1.5), 2), "routing": rng.randrange(1 << 20)}
        if op == "grouped":
            case["dtype"] = "fp8" if fp8 else "bf16"
            case["swiglu"] = swiglu
        if experts * max(_lengths(case)) * (k + columns) > 1.5e9:
            continue
        return case


def _lengths(case):
    """Rows of each expert: a draw of `t` rows over experts whose popularity spreads by `skew`."""
    r = np.random.RandomState(case["routing"])
    p = np.exp(case["skew"] * r.standard_normal(case["experts"]))
    return [int(v) for v in r.multinomial(case["t"], p / p.sum())]


def work(case):
    if case["op"] == "quantize":
        size = case["m"] * case["k"] * max(1, case["experts"])
        kb = -(-case["k"] // BLOCK)
        scales = (case["experts"] * -(-case["m"] // BLOCK) if case["experts"] else case["m"]) * kb
        return {"bytes": size * ((2 if case["dtype"] == "bf16" else 4) + 1) + 4 * scales,
                "flops": 2 * size}
    n, k = case["n"], case["k"]
    if case["op"] == "backward":
        t, lengths = case["t"], _lengths(case)
        used = sum(1 for v in lengths if v)
        bytes_ = 2 * (2 * t * k + t * n + used * n * k + len(lengths) * n * k)
        return {"bytes": bytes_ + 4 * (len(lengths) + 1), "flops": 4.0 * t * n * k}
    columns = 2 * n if case["swiglu"] else n
    if case["op"] == "fp8":
        t, used, offsets, fp8 = case["m"], 1, 0, True
    else:
        lengths = _lengths(case)
        t, used, offsets = case["t"], sum(1 for v in lengths if v), len(lengths) + 1
        fp8 = case["dtype"] == "fp8"
    bytes_ = (t * k + used * columns * k) * (1 if fp8 else 2) + 2 * t * n + 4 * offsets
    if fp8:
        kb = -(-k // BLOCK)
        bytes_ += 4 * kb * (t + used * -(-columns // BLOCK))
    return {"bytes": bytes_, "flops": 2.0 * t * columns * k}


# ------------------------------------------------------------------ inputs


def _activations(shape, g):
    """Normal rows with channels of different spread, a few of them large, as hidden states have."""
    k = shape[-1]
    channel = torch.exp(0.5 * torch.randn(k, generator=g, device="cuda"))
    channel[torch.randint(0, k, (max(1, k // 500),), generator=g, device="cuda")] *= 10.0
    return torch.randn(shape, generator=g, device="cuda") * channel


def _weights(shape, g):
    return torch.randn(shape, generator=g, device="cuda") * shape[-1] ** -0.5


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    state = dict(case)
    if case["op"] == "quantize":
        if case["experts"]:
            x = _weights((case["experts"], case["m"], case["k"]), g)
        else:
            x = _activations((case["m"], case["k"]), g)
        state["x"] = x.to(DTYPES[case["dtype"]])
        return state
    n, k = case["n"], case["k"]
    columns = 2 * n if case.get("swiglu") else n
    if case["op"] == "fp8":
        state["x"], state["xs"] = _quantize_rows(_activations((case["m"], k), g).bfloat16())
        state["w"], state["ws"] = _quantize_tiles(_weights((columns, k), g)[None])
        state["w"], state["ws"] = state["w"][0], state["ws"][0]
        return state
    lengths = _lengths(case)
    random.Random(seed).shuffle(lengths)  # which expert has how many rows
    offsets = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
    state["offsets"] = torch.from_numpy(offsets).cuda()
    # the plan of the padded plain form: a row number for each expert's slots,
    # t (a row of zeros) where an expert has fewer rows; and each row's slot
    longest = max(1, max(lengths))
    slot = np.arange(longest)[None, :]
    rows = offsets[:-1, None] + slot
    rows = np.where(slot < np.array(lengths)[:, None], rows, case["t"]).reshape(-1)
    state["rows"] = torch.from_numpy(rows.astype(np.int64)).cuda()
    state["slots"] = torch.from_numpy(np.flatnonzero(rows < case["t"])).cuda()
    x = _activations((case["t"], k), g).bfloat16()
    w = _weights((case["experts"], columns, k), g).bfloat16()
    if case["op"] == "backward":
        state["x"], state["w"] = x, w
        state["grad"] = (torch.randn((case["t"], n), generator=g, device="cuda") * 1e-3).bfloat16()
    elif case["dtype"] == "fp8":
        state["x"], state["xs"] = _quantize_rows(x)
        state["w"], state["ws"] = _quantize_tiles(w)
    else:
        state["x"], state["w"] = x, w
    return state


# ------------------------------------------------------------------ plain forms


def _to_e4m3(x, inverse):
    return (x * inverse).clamp(-E4M3_MAX, E4M3_MAX).to(F8)


def _quantize_rows(x):
    """[m, k] to e4m3 values and one fp32 scale for each 128 columns of a row."""
    m, k = x.shape
    kb = -(-k // BLOCK)
    v = torch.zeros((m, kb * BLOCK), device=x.device, dtype=torch.float32)
    v[:, :k] = x
    v = v.view(m, kb, BLOCK)
    amax = v.abs().amax(2).clamp(min=AMAX_FLOOR)
    q = _to_e4m3(v, (E4M3_MAX / amax)[:, :, None])
    return q.view(m, kb * BLOCK)[:, :k].contiguous(), amax / E4M3_MAX


def _quantize_tiles(w):
    """[e, n, k] to e4m3 values and one fp32 scale for each 128 x 128 tile."""
    e, n, k = w.shape
    nb, kb = -(-n // BLOCK), -(-k // BLOCK)
    v = torch.zeros((e, nb * BLOCK, kb * BLOCK), device=w.device, dtype=torch.float32)
    v[:, :n, :k] = w
    v = v.view(e, nb, BLOCK, kb, BLOCK)
    amax = v.abs().amax((2, 4)).clamp(min=AMAX_FLOOR)
    q = _to_e4m3(v, (E4M3_MAX / amax)[:, :, None, :, None])
    return q.view(e, nb * BLOCK, kb * BLOCK)[:, :n, :k].contiguous(), amax / E4M3_MAX


def _rows_from(q, scale):
    return q.float() * scale.repeat_interleave(BLOCK, 1)[:, : q.shape[1]]


def _tiles_from(q, scale):
    n, k = q.shape[-2:]
    s = scale.repeat_interleave(BLOCK, -2)[..., :n, :].repeat_interleave(BLOCK, -1)[..., :k]
    return q.float() * s


def _swiglu(h):
    n = h.shape[-1] // 2
    gate, up = h[..., :n], h[..., n:]
    return gate / (1.0 + torch.exp(-gate)) * up


def _by_expert(state, v):
    """Rows sorted by expert as [experts, longest, width], zeros in the slots that have no row."""
    v = torch.cat([v, torch.zeros_like(v[:1])]) if v.shape[0] else v.new_zeros((1, v.shape[1]))
    return v[state["rows"]].view(state["experts"], -1, v.shape[1])


def _in_order(state, v):
    """The other way: each row's slot of [experts, longest, width]."""
    return v.reshape(-1, v.shape[2])[state["slots"]]


def run(state):
    op = state["op"]
    if own:
        fp8, grouped = _library()
        if op == "quantize":
            if state["experts"]:
                return fp8.quantize_fp8_block128_weight(state["x"])
            return fp8.quantize_fp8_block128(state["x"])
        if op == "fp8":
            gemm = fp8.gemm_swiglu_fp8_block128 if state["swiglu"] else fp8.gemm_fp8_block128
            return gemm(state["x"], state["xs"], state["w"], state["ws"])
        if op == "backward":
            return grouped.gemm_grouped_bf16_backward(state["grad"], state["x"], state["w"],
                                                      state["offsets"])
        if state["dtype"] == "fp8":
            gemm = (grouped.gemm_grouped_swiglu_fp8_block128 if state["swiglu"]
                    else grouped.gemm_grouped_fp8_block128)
            return gemm(state["x"], state["xs"], state["w"], state["ws"], state["offsets"])
        gemm = grouped.gemm_grouped_swiglu_bf16 if state["swiglu"] else grouped.gemm_grouped_bf16
        return gemm(state["x"], state["w"], state["offsets"])
    if op == "quantize":
        return _quantize_tiles(state["x"]) if state["experts"] else _quantize_rows(state["x"])
    if op == "fp8":
        h = _rows_from(state["x"], state["xs"]) @ _tiles_from(state["w"], state["ws"]).t()
        return (_swiglu(h) if state["swiglu"] else h).bfloat16()
    if op == "backward":
        grad = _by_expert(state, state["grad"].float())
        dx = _in_order(state, grad @ state["w"].float())
        dw = grad.transpose(1, 2) @ _by_expert(state, state["x"].float())
        return dx.bfloat16(), dw.bfloat16()
    if state["dtype"] == "fp8":
        x, w = _rows_from(state["x"], state["xs"]), _tiles_from(state["w"], state["ws"])
    else:
        x, w = state["x"].float(), state["w"].float()
    h = _in_order(state, _by_expert(state, x) @ w.transpose(1, 2))
    return (_swiglu(h) if state["swiglu"] else h).bfloat16()


# ------------------------------------------------------------------ 64 bits


def _grid_e4m3(v):
    """Values in [-448, 448] to the nearest of e4m3's: 3 bits behind the leading one, ties to even."""
    _, e = torch.frexp(v)
    step = torch.pow(2.0, (e.clamp(min=-5) - 4).double())
    return torch.round(v / step) * step


def _blocks64(v, height):
    """Scale (64 bits) of each height x 128 block, and it spread over the values."""
    n, k = v.shape
    rows = torch.arange(n, device=v.device) // height
    cols = torch.arange(k, device=v.device) // BLOCK
    nb, kb = -(-n // height), -(-k // BLOCK)
    flat = (rows[:, None] * kb + cols[None, :]).reshape(-1)
    amax = torch.full((nb * kb,), AMAX_FLOOR, dtype=torch.float64, device=v.device)
    amax = amax.scatter_reduce(0, flat, v.abs().reshape(-1), "amax")
    return (amax / 448.0).view(nb, kb), amax[flat].view(n, k)


def _spread64(scale, height, n, k):
    rows = torch.arange(n, device=scale.device) // height
    cols = torch.arange(k, device=scale.device) // BLOCK
    return scale.double()[rows][:, cols]


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        parts, height = (state["x"], BLOCK) if case["experts"] else (state["x"][None], 1)
        q, s = [], []
        for part in parts:
            v = part.double()
            scale, amax = _blocks64(v, height)
            q.append(_grid_e4m3(v * 448.0 / amax))
            s.append(scale)
        return (torch.stack(q), torch.stack(s)) if case["experts"] else (q[0], s[0])
    n, k = case["n"], case["k"]
    columns = 2 * n if case.get("swiglu") else n
    if op == "fp8":
        ranges, weights, scales = [(0, case["m"])], state["w"][None], state["ws"][None]
    else:
        ends = state["offsets"].tolist()
        ranges, weights, scales = list(zip(ends[:-1], ends[1:])), state["w"], state.get("ws")
    rows = state["x"].shape[0]
    if op == "backward":
        dx = torch.zeros((rows, k), dtype=torch.float64, device="cuda")
        dw = torch.zeros((case["experts"], n, k), dtype=torch.float64, device="cuda")
        for e, (a, b) in enumerate(ranges):
            grad = state["grad"][a:b].double()
            dx[a:b] = torch.matmul(grad, weights[e].double())
            dw[e] = torch.matmul(grad.mT, state["x"][a:b].double())
        return dx, dw
    out = torch.zeros((rows, n), dtype=torch.float64, device="cuda")
    for e, (a, b) in enumerate(ranges):
        if a == b:
            continue
        x, w = state["x"][a:b].double(), weights[e].double()
        if scales is not None:
            x *= _spread64(state["xs"][a:b], 1, b - a, k)
            w *= _spread64(scales[e], BLOCK, columns, k)
        h = torch.matmul(x, w.mT)
        out[a:b] = h[:, :n] * torch.sigmoid(h[:, :n]) * h[:, n:] if case["swiglu"] else h
    return out
