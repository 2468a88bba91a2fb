"""Each tile shape of the expert-layer products against 64-bit forms (GPU).

Tolerances are those of expert_math (derived there).
"""

from __future__ import annotations

import pytest
import torch

import expert_math as em
from conftest import seeded
from cuda_operator_lab import bindings as b
from cuda_operator_lab import grouped

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rows_of(lengths):
    ends = em.offsets_of(lengths).tolist()
    return [(e, slice(lo, hi)) for e, (lo, hi) in enumerate(zip(ends[:-1], ends[1:]))]


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
