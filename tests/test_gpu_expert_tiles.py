"""Each tile shape of the expert-layer products against 64-bit forms (GPU).

Tolerances are those of expert_math (derived there).
"""

from __future__ import annotations

import json
import subprocess
import sys

import pytest
import torch

import expert_math as em
import expert_tiles as et
from conftest import PACKAGE_DIR, seeded
from cuda_operator_lab import bindings as b
from cuda_operator_lab import fp8, grouped

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rows_of(lengths):
    ends = em.offsets_of(lengths).tolist()
    return [(e, slice(lo, hi)) for e, (lo, hi) in enumerate(zip(ends[:-1], ends[1:]))]


def on_148_sms():
    return b.device_info()["sm_count"] == et.SM_COUNT


@pytest.mark.parametrize("product,tiles,t,experts,n,k", et.CASES)
def test_each_tile_shape(product, tiles, t, experts, n, k):
    if on_148_sms():
        assert b.expert_tiles(product, t, k, n, experts) == tiles
    g = seeded(t + n + k)
    lengths = et.ragged(t, experts)
    off = em.offsets_of(lengths).to(DEV)
    swiglu = "swiglu" in product
    x = (torch.randn(t, k, generator=g) * torch.exp(torch.randn(k, generator=g))).bfloat16().to(DEV)
    grad = torch.randn(t, n, generator=g).bfloat16().to(DEV)
    w = (torch.randn(experts, 2 * n if swiglu else n, k, generator=g) * k ** -0.5).bfloat16().to(DEV)
    if "fp8" in product:
        xq, xs = fp8.quantize_fp8_block128(x)
        wq, ws = fp8.quantize_fp8_block128_weight(w)
        if product.startswith("dense"):
            gemm = fp8.gemm_swiglu_fp8_block128 if swiglu else fp8.gemm_fp8_block128
            call = lambda: (gemm(xq, xs, wq[0], ws[0]),)  # noqa: E731
        else:
            gemm = grouped.gemm_grouped_swiglu_fp8_block128 if swiglu else grouped.gemm_grouped_fp8_block128
            call = lambda: (gemm(xq, xs, wq, ws, off),)  # noqa: E731
        xd, wd = xq.double() * em.spread(xs, 1, t, k), wq.double() * em.spread(ws, 128, *w.shape[1:])
        wanted = [lambda e, r: em.product(xd[r], wd[e], swiglu)]
    else:
        by_x = lambda e, r: em.product(grad[r].double(), w[e].double().mT, False)  # noqa: E731
        by_w = lambda e, r: em.product(grad[r].double().mT, x[r].double().mT, False)  # noqa: E731
        call, wanted = {
            "bf16": (lambda: (grouped.gemm_grouped_bf16(x, w, off),),
                     [lambda e, r: em.product(x[r].double(), w[e].double(), False)]),
            "swiglu_bf16": (lambda: (grouped.gemm_grouped_swiglu_bf16(x, w, off),),
                            [lambda e, r: em.product(x[r].double(), w[e].double(), True)]),
            "grad_input": (lambda: (grouped.gemm_grouped_bf16_grad_input(grad, w, off),), [by_x]),
            "grad_weight": (lambda: (grouped.gemm_grouped_bf16_grad_weight(grad, x, off),), [by_w]),
            "both_grads": (lambda: grouped.gemm_grouped_bf16_backward(grad, x, w, off), [by_x, by_w]),
        }[product]
    got = call()
    assert b.gemm_status() == 0
    for y, want in zip(got, wanted):
        of_experts = y.ndim == 3
        for e, r in rows_of(lengths):
            em.assert_within(y[e] if of_experts else y[r], *want(e, r))
    again = call()
    assert all(torch.equal(p, q) for p, q in zip(got, again))


def test_first_calls_of_each_set_up_inside_a_capture():
    """Pairs ask how many fit the device and the wide e4m3 tiles how many registers they
    start with, on their first call: it may be one that is captured."""
    cases = [c for c in et.CASES if c[1] in (et.PAIRS, et.WIDE) and c[0] in
             ("bf16", "swiglu_bf16", "grad_input", "grad_weight", "fp8", "swiglu_fp8", "dense_fp8")]
    code = """
import json, sys, torch
sys.path.insert(0, sys.argv[1])
from cuda_operator_lab import bindings, fp8, grouped
E4M3 = torch.float8_e4m3fn
prepared = []
for product, t, experts, n, k, lengths in json.loads(sys.argv[2]):
    rows = 2 * n if "swiglu" in product else n
    off = torch.tensor([0] + lengths, dtype=torch.int32).cumsum(0).int().cuda()
    if "fp8" in product:
        kb, nb = -(-k // 128), -(-rows // 128)
        x, w = torch.ones(t, k, device="cuda").to(E4M3), torch.ones(experts, rows, k, device="cuda").to(E4M3)
        xs, ws = torch.full((t, kb), 0.5, device="cuda"), torch.full((experts, nb, kb), 0.5, device="cuda")
        if product == "dense_fp8":
            call = lambda a=(x, xs, w[0], ws[0]): fp8.gemm_fp8_block128(*a)
        else:
            f = grouped.gemm_grouped_swiglu_fp8_block128 if rows != n else grouped.gemm_grouped_fp8_block128
            call = lambda f=f, a=(x, xs, w, ws, off): f(*a)
        total, want = k / 4, None
    else:
        x = torch.ones(t, k, device="cuda", dtype=torch.bfloat16)
        g = torch.ones(t, n, device="cuda", dtype=torch.bfloat16)
        w = torch.ones(experts, rows, k, device="cuda", dtype=torch.bfloat16)
        total, want = float(k), None
        if product == "grad_input":
            total, call = float(n), lambda a=(g, w, off): grouped.gemm_grouped_bf16_grad_input(*a)
        elif product == "grad_weight":
            want = torch.tensor(lengths).bfloat16().view(-1, 1, 1)
            call = lambda a=(g, x, off): grouped.gemm_grouped_bf16_grad_weight(*a)
        elif rows != n:
            call = lambda a=(x, w, off): grouped.gemm_grouped_swiglu_bf16(*a)
        else:
            call = lambda a=(x, w, off): grouped.gemm_grouped_bf16(*a)
    if want is None:  # silu(s) is s in bf16 for sums this large
        want = torch.tensor(total * total if rows != n else total).bfloat16()
    prepared.append((product, call, want.cuda()))
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    outs = [call() for _, call, _ in prepared]
graph.replay()
torch.cuda.synchronize()
for (product, _, want), y in zip(prepared, outs):
    assert (y == want).all(), product
assert bindings.gemm_status() == 0
print("captured")
"""
    sizes = [(p, t, experts, n, k, et.ragged(t, experts)) for p, _, t, experts, n, k in cases]
    done = subprocess.run([sys.executable, "-c", code, str(PACKAGE_DIR), json.dumps(sizes)],
                          capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "captured" in done.stdout, done.stdout + done.stderr


@pytest.mark.parametrize("lengths", [
    # ends inside a step of 16 rows, on one, one row over, an expert without rows
    [1003, 977, 0, 1024, 1041, 993, 1008, 1025],
    # more and shorter experts: a worker's tiles end every dozen blocks
    [645 + 11 * (i % 13) for i in range(12)],
])
def test_weight_gradient_of_cta_pairs(lengths):
    """Both CTAs of a pair zero the rows behind a ragged tail in their own shared
    memory; the MMAs that one of them issues read both.  The row behind each
    expert's last one is another expert's, and large, so that a row not zeroed shows."""
    n, k, t = 2048, 2048, sum(lengths)
    g = seeded(t)
    off = em.offsets_of(lengths).to(DEV)
    x = torch.randn(t, k, generator=g).bfloat16()
    grad = torch.randn(t, n, generator=g).bfloat16()
    for _, r in rows_of(lengths):
        x[r][:16] *= 64
        grad[r][:16] *= 64
    x, grad = x.to(DEV), grad.to(DEV)
    dw = grouped.gemm_grouped_bf16_grad_weight(grad, x, off)
    assert b.gemm_status() == 0
    for e, r in rows_of(lengths):
        em.assert_within(dw[e], *em.product(grad[r].double().mT, x[r].double().mT, False))
    for _ in range(5):
        assert torch.equal(grouped.gemm_grouped_bf16_grad_weight(grad, x, off), dw)
    assert b.gemm_status() == 0


def test_sums_of_seconds_end_by_themselves():
    """An expert of 3/4 of 2**30 rows: one CTA sums its only tile for seconds, its
    warps that store it and that zero the next ragged tail wait all that time.  The
    CTA's next tile is that of expert 148, whose 17 rows end inside a step of 16."""
    many, n, k = 3 << 28, 8, 8
    lengths = [many] + [0] * 147 + [17, 5]
    t, off = sum(lengths), em.offsets_of(lengths).to(DEV)
    g = seeded(90)
    x = torch.zeros(t, k, device=DEV, dtype=torch.bfloat16)
    grad = torch.zeros(t, n, device=DEV, dtype=torch.bfloat16)
    some = torch.randint(0, many, (200,), generator=g).unique()
    some = torch.cat([some, torch.tensor([many - 1]), torch.arange(many, t)]).unique()
    xs = em.small_integers((len(some), k), g, 1)
    gs = em.small_integers((len(some), n), g, 1)
    x[some.to(DEV)] = xs.bfloat16().to(DEV)
    grad[some.to(DEV)] = gs.bfloat16().to(DEV)
    dw = grouped.gemm_grouped_bf16_grad_weight(grad, x, off)
    assert b.gemm_status() == 0
    del x, grad
    dw = dw.float().cpu()
    for e, lo, hi in ((0, 0, many), (148, many, many + 17), (149, many + 17, t)):
        mine = (some >= lo) & (some < hi)
        assert torch.equal(dw[e], gs[mine].t() @ xs[mine])
    assert not dw[1:148].any()
