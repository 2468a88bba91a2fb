"""Products grouped by expert and their gradients against 64-bit forms (GPU).

Tolerances are those of expert_math (derived there).  Sums of small integers
are exact in every type on the way, so most checks there are of equality.
"""

from __future__ import annotations

import subprocess
import sys

import pytest
import torch

import expert_math as em
from conftest import PACKAGE_DIR, seeded
from cuda_operator_lab import bindings as b
from cuda_operator_lab import fp8, grouped

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3 = torch.float8_e4m3fn

#: Rows of each expert: none, one, odd counts, several tiles, one that takes all.
LENGTHS = {
    "one": [1],
    "ones": [1, 1, 1, 1, 1],
    "gaps": [0, 3, 0, 0, 17, 0],
    "ragged": [130, 0, 1, 255, 64, 7],
    "edges": [128, 256, 127, 129, 64, 63, 65],
    "all in one": [0, 0, 700, 0],
    "nothing": [0, 0, 0],
    "many": [(5 * i) % 11 for i in range(100)],
}
SIZES = [(8, 8), (64, 64), (72, 136), (264, 200), (520, 392)]


def groups(lengths):
    ends = em.offsets_of(lengths).tolist()
    return list(zip(ends[:-1], ends[1:]))


def bf(t):
    return t.to(torch.bfloat16).to(DEV)


@pytest.mark.parametrize("name", LENGTHS)
@pytest.mark.parametrize("n,k", SIZES + [(129, 72), (77, 40), (50, 37), (33, 1)])
def test_forward_of_small_integers_is_exact(name, n, k):
    lengths = LENGTHS[name]
    g = seeded(n * 1000 + k)
    x = em.small_integers((sum(lengths), k), g, 1)
    w = em.small_integers((len(lengths), n, k), g, 1)
    w[:, :, 48:] *= (torch.rand(w[:, :, 48:].shape, generator=g) < 0.3)  # keeps sums under 256
    y = grouped.gemm_grouped_bf16(bf(x), bf(w), em.offsets_of(lengths).to(DEV))
    assert b.gemm_status() == 0
    for e, (lo, hi) in enumerate(groups(lengths)):
        assert torch.equal(y[lo:hi].float().cpu(), x[lo:hi] @ w[e].t()), e


@pytest.mark.parametrize("name", LENGTHS)
@pytest.mark.parametrize("n,k", SIZES + [(129, 72), (50, 37)])
def test_forward_swiglu(name, n, k):
    lengths = LENGTHS[name]
    g = seeded(n * 1000 + k + 1)
    x = torch.randn(sum(lengths), k, generator=g).bfloat16()
    w = (torch.randn(len(lengths), 2 * n, k, generator=g) * k ** -0.5).bfloat16()
    y = grouped.gemm_grouped_swiglu_bf16(x.to(DEV), w.to(DEV), em.offsets_of(lengths).to(DEV))
    assert b.gemm_status() == 0
    for e, (lo, hi) in enumerate(groups(lengths)):
        em.assert_within(y[lo:hi].cpu(), *em.product(x[lo:hi].double(), w[e].double(), True))


# One size at least for each tile shape that the library chooses from: few rows
# an expert, half-filled tiles, several whole ones.
TILES = [([300, 513, 0, 129], 136, 144), ([300, 513, 0, 129], 2000, 144),
         ([300, 513, 0, 129], 136, 2064), ([700, 0, 650], 2000, 2064), ([700, 0, 650], 1000, 2064),
         ([100] * 16, 136, 144), ([90, 70, 0, 110, 128, 60], 1000, 528),
         ([20] * 10, 264, 2064), ([5, 0, 40, 3], 264, 2064),
         # gradients whose sums the CTAs of a cluster share
         ([5, 0, 40, 3], 1032, 136), ([20] * 10, 1032, 264), ([1, 0, 1], 4104, 520)]


def pairs_of(lengths):
    return [(e, slice(lo, hi)) for e, (lo, hi) in enumerate(groups(lengths))]


@pytest.mark.parametrize("lengths,n,k", TILES)
def test_tile_shapes_bf16(lengths, n, k):
    g = seeded(n + k + len(lengths))
    t, off = sum(lengths), em.offsets_of(lengths).to(DEV)
    x = torch.randn(t, k, generator=g).bfloat16().to(DEV)
    grad = torch.randn(t, n, generator=g).bfloat16().to(DEV)
    w = (torch.randn(len(lengths), 2 * n, k, generator=g) * k ** -0.5).bfloat16().to(DEV)
    one = w[:, :n].contiguous()
    y, h = grouped.gemm_grouped_bf16(x, one, off), grouped.gemm_grouped_swiglu_bf16(x, w, off)
    dx, dw = grouped.gemm_grouped_bf16_backward(grad, x, one, off)
    assert b.gemm_status() == 0
    for e, r in pairs_of(lengths):
        xr, gr, we = x[r].double(), grad[r].double(), w[e].double()
        em.assert_within(y[r], *em.product(xr, we[:n], False))
        em.assert_within(h[r], *em.product(xr, we, True))
        em.assert_within(dx[r], *em.product(gr, we[:n].mT, False))
        em.assert_within(dw[e], *em.product(gr.mT, xr.mT, False))


def test_tile_shapes_of_long_batches():
    """Thousands of rows an expert: the widest tiles of all four products."""
    lengths, n, k = [2001, 1950, 0, 2300], 1032, 2048
    g = seeded(21)
    t, off = sum(lengths), em.offsets_of(lengths).to(DEV)
    x = torch.randn(t, k, generator=g).bfloat16().to(DEV)
    grad = torch.randn(t, n, generator=g).bfloat16().to(DEV)
    w = (torch.randn(4, n, k, generator=g) * k ** -0.5).bfloat16().to(DEV)
    y = grouped.gemm_grouped_bf16(x, w, off)
    dx, dw = grouped.gemm_grouped_bf16_backward(grad, x, w, off)
    xq, xs, wq, ws = quantized(x, w)
    y8 = grouped.gemm_grouped_fp8_block128(xq, xs, wq, ws, off)
    assert b.gemm_status() == 0
    xd, wd = xq.double() * em.spread(xs, 1, t, k), wq.double() * em.spread(ws, 128, n, k)
    for e, r in pairs_of(lengths):
        xr, gr, we = x[r].double(), grad[r].double(), w[e].double()
        em.assert_within(y[r], *em.product(xr, we, False))
        em.assert_within(dx[r], *em.product(gr, we.mT, False))
        em.assert_within(dw[e], *em.product(gr.mT, xr.mT, False))
        em.assert_within(y8[r], *em.product(xd[r], wd[e], False))


@pytest.mark.parametrize("lengths,n,k", TILES + [([300, 513, 0, 129], 136, 528),
                                                 ([20] * 10, 136, 2064), ([20] * 10, 264, 528),
                                                 ([100] * 16, 1000, 144),
                                                 ([90, 70, 0, 110, 128, 60], 136, 528),
                                                 ([5, 0, 40, 3], 136, 2064)])
@pytest.mark.parametrize("swiglu", [False, True])
def test_tile_shapes_fp8(lengths, n, k, swiglu):
    n = -(-n // 128) * 128 if swiglu else n
    g = seeded(n + k + len(lengths))
    x = torch.randn(sum(lengths), k, generator=g) * torch.exp(torch.randn(k, generator=g))
    w = torch.randn(len(lengths), 2 * n if swiglu else n, k, generator=g) * k ** -0.5
    xq, xs, wq, ws = quantized(x, w)
    gemm = grouped.gemm_grouped_swiglu_fp8_block128 if swiglu else grouped.gemm_grouped_fp8_block128
    y = gemm(xq, xs, wq, ws, em.offsets_of(lengths).to(DEV))
    assert b.gemm_status() == 0
    xd, wd = xq.double() * em.spread(xs, 1, *x.shape), wq.double() * em.spread(ws, 128, *w.shape[1:])
    for e, r in pairs_of(lengths):
        em.assert_within(y[r], *em.product(xd[r], wd[e], swiglu))


@pytest.mark.parametrize("lengths", [[5, 0, 40, 3], [300, 513, 0, 129], [2] * 48])
@pytest.mark.parametrize("n,k", [(1000, 2048), (384, 4104)])
def test_forward_of_long_sums(lengths, n, k):
    g = seeded(n + k)
    x = torch.randn(sum(lengths), k, generator=g).bfloat16()
    w = (torch.randn(len(lengths), n, k, generator=g) * k ** -0.5).bfloat16()
    y = grouped.gemm_grouped_bf16(x.to(DEV), w.to(DEV), em.offsets_of(lengths).to(DEV))
    assert b.gemm_status() == 0
    for e, (lo, hi) in enumerate(groups(lengths)):
        em.assert_within(y[lo:hi].cpu(), *em.product(x[lo:hi].double(), w[e].double(), False))


@pytest.mark.parametrize("name", LENGTHS)
@pytest.mark.parametrize("n,k", SIZES + [(40, 77), (37, 50), (1, 33)])
def test_backward_of_small_integers_is_exact(name, n, k):
    lengths = LENGTHS[name]
    t = sum(lengths)
    g = seeded(n * 1000 + k + 2)
    x = em.small_integers((t, k), g, 1)
    w = em.small_integers((len(lengths), n, k), g, 1)
    grad = em.small_integers((t, n), g, 1)
    w *= (torch.rand(w.shape, generator=g) < 0.3)     # keeps sums under 256
    x *= (torch.rand(x.shape, generator=g) < 0.3)
    dx, dw = grouped.gemm_grouped_bf16_backward(bf(grad), bf(x), bf(w),
                                                em.offsets_of(lengths).to(DEV))
    assert b.gemm_status() == 0
    assert dx.shape == (t, k) and dw.shape == w.shape
    for e, (lo, hi) in enumerate(groups(lengths)):
        assert torch.equal(dx[lo:hi].float().cpu(), grad[lo:hi] @ w[e]), e
        assert torch.equal(dw[e].float().cpu(), grad[lo:hi].t() @ x[lo:hi]), e


@pytest.mark.parametrize("lengths", [[700, 0, 31, 1500], [16, 15, 17, 1, 0, 48]])
def test_backward_of_long_sums(lengths):
    n, k, t = 520, 1032, sum(lengths)
    g = seeded(t)
    x, grad = (torch.randn(t, c, generator=g).bfloat16() for c in (k, n))
    w = torch.randn(len(lengths), n, k, generator=g).bfloat16()
    dx, dw = grouped.gemm_grouped_bf16_backward(grad.to(DEV), x.to(DEV), w.to(DEV),
                                                em.offsets_of(lengths).to(DEV))
    assert b.gemm_status() == 0
    for e, (lo, hi) in enumerate(groups(lengths)):
        gr, xr = grad[lo:hi].double(), x[lo:hi].double()
        em.assert_within(dx[lo:hi].cpu(), *em.product(gr, w[e].double().mT, False))
        em.assert_within(dw[e].cpu(), *em.product(gr.mT, xr.mT, False))


@pytest.mark.parametrize("lengths,n,k", [([3, 0, 9, 2], 184, 216), ([200, 31, 0], 320, 200),
                                         ([70, 0, 5, 130] * 5, 776, 520), ([2] * 60, 384, 160),
                                         ([400, 333, 64], 2000, 1032), ([0, 0], 64, 64)])
def test_both_gradients_are_those_of_their_own_calls(lengths, n, k):
    """In one launch side by side or after one another; some rows of no expert."""
    t, off = sum(lengths) + 9, em.offsets_of(lengths, 4).to(DEV)
    g = seeded(t)
    x, grad = em.small_integers((t, k), g, 1), em.small_integers((t, n), g, 1)
    w = em.small_integers((len(lengths), n, k), g, 1)
    x *= (torch.rand(x.shape, generator=g) < 0.2)
    w *= (torch.rand(w.shape, generator=g) < 0.05)
    grad[:, 100:] *= (torch.rand(grad[:, 100:].shape, generator=g) < 0.2)
    dx, dw = grouped.gemm_grouped_bf16_backward(bf(grad), bf(x), bf(w), off)
    used = slice(4, 4 + sum(lengths))
    assert torch.equal(dx[used], grouped.gemm_grouped_bf16_grad_input(bf(grad), bf(w), off)[used])
    assert torch.equal(dw, grouped.gemm_grouped_bf16_grad_weight(bf(grad), bf(x), off))
    assert b.gemm_status() == 0
    ends = off.tolist()
    for e, (lo, hi) in enumerate(zip(ends[:-1], ends[1:])):
        assert torch.equal(dx[lo:hi].float().cpu(), grad[lo:hi] @ w[e])
        assert torch.equal(dw[e].float().cpu(), grad[lo:hi].t() @ x[lo:hi])


def test_gradients_against_differences():
    """The forward product is linear in x and in W, so a difference of any size
    is the gradient's product with it; in small integers both are exact."""
    lengths, n, k = [40, 0, 65, 3], 64, 48
    t, off = sum(lengths), em.offsets_of(lengths).to(DEV)
    g = seeded(20)
    x, dx_step = (em.small_integers((t, k), g, 1) for _ in range(2))
    w, dw_step = (em.small_integers((len(lengths), n, k), g, 1) for _ in range(2))
    grad = em.small_integers((t, n), g, 1)
    gx, gw = grouped.gemm_grouped_bf16_backward(bf(grad), bf(x), bf(w), off)

    def loss(xv, wv):
        return float((grouped.gemm_grouped_bf16(bf(xv), bf(wv), off).double().cpu() * grad.double()).sum())

    base = loss(x, w)
    assert loss(x + dx_step, w) - base == float((gx.double().cpu() * dx_step.double()).sum())
    assert loss(x, w + dw_step) - base == float((gw.double().cpu() * dw_step.double()).sum())


def quantized(x, w):
    return (*fp8.quantize_fp8_block128(x.to(DEV)), *fp8.quantize_fp8_block128_weight(w.to(DEV)))


@pytest.mark.parametrize("name", LENGTHS)
@pytest.mark.parametrize("n,k,swiglu", [(16, 16, False), (136, 272, False), (129, 512, False),
                                        (520, 1040, False), (128, 144, True), (384, 512, True),
                                        (128, 100, True), (70, 77, False)])
def test_fp8(name, n, k, swiglu):
    lengths = LENGTHS[name]
    g = seeded(n * 1000 + k + 3)
    x = torch.randn(sum(lengths), k, generator=g) * torch.exp(torch.randn(k, generator=g))
    w = torch.randn(len(lengths), 2 * n if swiglu else n, k, generator=g) * k ** -0.5
    xq, xs, wq, ws = quantized(x, w)
    gemm = grouped.gemm_grouped_swiglu_fp8_block128 if swiglu else grouped.gemm_grouped_fp8_block128
    y = gemm(xq, xs, wq, ws, em.offsets_of(lengths).to(DEV))
    assert b.gemm_status() == 0
    xd, wd = xq.double() * em.spread(xs, 1, *x.shape), wq.double() * em.spread(ws, 128, *w.shape[1:])
    for e, (lo, hi) in enumerate(groups(lengths)):
        em.assert_within(y[lo:hi], *em.product(xd[lo:hi], wd[e], swiglu))


# ---------------------------------------------------------------- rows of no expert


@pytest.mark.parametrize("first,lengths,after", [(0, [5, 70, 0], 60), (9, [130, 3], 1),
                                                 (64, [0, 0], 64), (3, [257], 0)])
def test_rows_of_no_expert_are_neither_used_nor_written(first, lengths, after):
    n, k = 136, 72
    t = first + sum(lengths) + after
    off = em.offsets_of(lengths, first).to(DEV)
    used = torch.zeros(t, dtype=torch.bool)
    used[first:first + sum(lengths)] = True
    g = seeded(t)
    x, grad = em.small_integers((t, k), g, 1), em.small_integers((t, n), g, 1)
    w = em.small_integers((len(lengths), n, k), g, 1)
    spoiled_x, spoiled_grad = x.clone(), grad.clone()
    spoiled_x[~used], spoiled_grad[~used] = float("nan"), float("inf")
    y = torch.full((t, n), 7.0, device=DEV, dtype=torch.bfloat16)
    grouped.gemm_grouped_bf16_into(bf(spoiled_x), bf(w), off, y)
    dx = torch.full((t, k), 7.0, device=DEV, dtype=torch.bfloat16)
    grouped.gemm_grouped_bf16_grad_input_into(bf(spoiled_grad), bf(w), off, dx)
    dw = grouped.gemm_grouped_bf16_grad_weight(bf(spoiled_grad), bf(spoiled_x), off)
    assert b.gemm_status() == 0
    ends = off.cpu().tolist()
    for e, (lo, hi) in enumerate(zip(ends[:-1], ends[1:])):
        assert torch.equal(y[lo:hi].float().cpu(), x[lo:hi] @ w[e].t())
        assert torch.equal(dx[lo:hi].float().cpu(), grad[lo:hi] @ w[e])
        assert torch.equal(dw[e].float().cpu(), grad[lo:hi].t() @ x[lo:hi])
    assert (y[~used.to(DEV)] == 7).all() and (dx[~used.to(DEV)] == 7).all()


def test_a_spoiled_expert_spoils_no_other():
    """NaN rows and weights of one expert: its neighbours' results do not change,
    although their tiles load some of its rows."""
    lengths, n, k = [70, 33, 100], 136, 72
    off = em.offsets_of(lengths).to(DEV)
    g = seeded(30)
    t = sum(lengths)
    x, grad = torch.randn(t, k, generator=g), torch.randn(t, n, generator=g)
    w = torch.randn(3, n, k, generator=g)
    y = grouped.gemm_grouped_bf16(bf(x), bf(w), off)
    dx, dw = grouped.gemm_grouped_bf16_backward(bf(grad), bf(x), bf(w), off)
    for t_ in (x[70:103], grad[70:103], w[1]):
        t_.fill_(float("nan"))
    y2 = grouped.gemm_grouped_bf16(bf(x), bf(w), off)
    dx2, dw2 = grouped.gemm_grouped_bf16_backward(bf(grad), bf(x), bf(w), off)
    for lo, hi, e in ((0, 70, 0), (103, 203, 2)):
        assert torch.equal(y2[lo:hi], y[lo:hi])
        assert torch.equal(dx2[lo:hi], dx[lo:hi])
        assert torch.equal(dw2[e], dw[e])
    assert torch.isnan(y2[70:103]).all() and torch.isnan(dw2[1]).all()


@pytest.mark.parametrize("wrong", [[-50, 10, 20, 30], [0, 40, 10, 60], [0, 10, 900, 2 ** 31 - 1],
                                   [500, 600, 700, 800], [-2 ** 31, -7, -3, -1]])
def test_wrong_offsets_stay_in_range(wrong):
    """What a wrong array gives is not defined, but nothing outside the tensors is touched."""
    t, n, k = 60, 72, 40
    off = torch.tensor(wrong, dtype=torch.int32, device=DEV)
    x, w, grad = (torch.randn(s, device=DEV).bfloat16() for s in ((t, k), (3, n, k), (t, n)))
    guard = 4096

    def guarded(*shape):
        size = 1
        for s in shape:
            size *= s
        whole = torch.full((size + 2 * guard,), 7.0, device=DEV, dtype=torch.bfloat16)
        return whole, whole[guard:guard + size].view(*shape)

    (ya, y), (dxa, dx), (dwa, dw), (y8a, y8) = guarded(t, n), guarded(t, k), guarded(3, n, k), guarded(t, n)
    grouped.gemm_grouped_bf16_into(x, w, off, y)
    grouped.gemm_grouped_bf16_grad_input_into(grad, w, off, dx)
    grouped.gemm_grouped_bf16_grad_weight_into(grad, x, off, dw)
    x8, w8 = x.repeat(1, 2)[:, :48].contiguous(), w.repeat(1, 1, 2)[:, :, :48].contiguous()
    grouped.gemm_grouped_fp8_block128_into(*quantized(x8, w8), off, y8)
    torch.cuda.synchronize()
    assert b.gemm_status() == 0
    for whole in (ya, dxa, dwa, y8a):
        assert (whole[:guard] == 7).all() and (whole[-guard:] == 7).all()


@pytest.mark.parametrize("wrong", [[-50, 10, 20, 30], [0, 40, 10, 60], [0, 10, 900, 2 ** 31 - 1],
                                   [7, 3, 50, 20], [500, 600, 700, 800], [-2 ** 31, -7, -3, -1]])
def test_offsets_count_as_the_largest_up_to_them(wrong):
    """Offsets that decrease or leave [0, T] act as their clamped running maximum:
    no row has two experts, rows of none are not written."""
    t, n, k = 60, 72, 48
    right = torch.tensor(wrong).clamp(0, t).cummax(0).values.int()
    g = seeded(35)
    x, grad = em.small_integers((t, k), g, 1), em.small_integers((t, n), g, 1)
    w = em.small_integers((3, n, k), g, 1)
    got, want = [], []
    for off, results in ((torch.tensor(wrong, dtype=torch.int32), got), (right, want)):
        off = off.to(DEV)
        for xs, ws, gs in ((bf(x), bf(w), bf(grad)), (bf(x[:, :-1]), bf(w[:, :-1, :-1]), bf(grad[:, :-1]))):
            y = torch.full((t, ws.shape[1]), 7.0, device=DEV, dtype=torch.bfloat16)
            dx = torch.full((t, ws.shape[2]), 7.0, device=DEV, dtype=torch.bfloat16)
            results.append(grouped.gemm_grouped_bf16_into(xs, ws, off, y))
            results.append(grouped.gemm_grouped_bf16_grad_input_into(gs, ws, off, dx))
            results.append(grouped.gemm_grouped_bf16_grad_weight(gs, xs, off))
    assert b.gemm_status() == 0
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    ends = right.tolist()
    for e, (lo, hi) in enumerate(zip(ends[:-1], ends[1:])):
        assert torch.equal(got[0][lo:hi].float().cpu(), x[lo:hi] @ w[e].t())
    assert (got[0][:ends[0]] == 7).all() and (got[0][ends[-1]:] == 7).all()


def test_most_experts():
    """1024 experts, most with a row or two, some with none."""
    experts, n, k = grouped.MAX_EXPERTS, 40, 24
    g = seeded(36)
    lengths = torch.randint(0, 4, (experts,), generator=g).tolist()
    t, off = sum(lengths), em.offsets_of(lengths).to(DEV)
    x, grad = em.small_integers((t, k), g, 1), em.small_integers((t, n), g, 1)
    w = em.small_integers((experts, n, k), g, 1)
    owner = torch.repeat_interleave(torch.arange(experts), torch.tensor(lengths))
    y = grouped.gemm_grouped_bf16(bf(x), bf(w), off)
    dx, dw = grouped.gemm_grouped_bf16_backward(bf(grad), bf(x), bf(w), off)
    assert b.gemm_status() == 0
    assert torch.equal(y.float().cpu(), torch.einsum("tk,tnk->tn", x, w[owner]))
    assert torch.equal(dx.float().cpu(), torch.einsum("tn,tnk->tk", grad, w[owner]))
    want = torch.zeros(experts, n, k).index_add_(0, owner, grad[:, :, None] * x[:, None, :])
    assert torch.equal(dw.float().cpu(), want)
    x8, w8 = torch.randn(t, 144, generator=g), torch.randn(experts, n, 144, generator=g)
    xq, xs, wq, ws = quantized(x8, w8)
    y8 = grouped.gemm_grouped_fp8_block128(xq, xs, wq, ws, off)
    xd, wd = xq.double() * em.spread(xs, 1, t, 144), wq.double() * em.spread(ws, 128, n, 144)
    own = owner.to(DEV)
    h = torch.einsum("tk,tnk->tn", xd, wd[own])
    err = (144 + 8) * 2.0 ** -23 * torch.einsum("tk,tnk->tn", xd.abs(), wd[own].abs())
    em.assert_within(y8, h, err + em.HALF_STEP_BF16 * (h.abs() + err))


def test_no_rows_at_all():
    w = torch.randn(2, 64, 32, device=DEV).bfloat16()
    off = torch.zeros(3, dtype=torch.int32, device=DEV)
    empty = torch.empty(0, 32, device=DEV, dtype=torch.bfloat16)
    grad = torch.empty(0, 64, device=DEV, dtype=torch.bfloat16)
    assert grouped.gemm_grouped_bf16(empty, w, off).shape == (0, 64)
    out = torch.full_like(w, 7)
    assert grouped.gemm_grouped_bf16_grad_weight_into(grad, empty, off, out) is out
    assert (out == 0).all()
    dx, dw = grouped.gemm_grouped_bf16_backward(grad, empty, w, off)
    assert dx.shape == (0, 32) and (dw == 0).all()


# ---------------------------------------------------------------- layouts, streams, graphs


def test_unaligned_operands():
    """Views two bytes off a 16-byte boundary, inputs and outputs."""
    lengths, n, k = [40, 0, 9], 72, 48
    off = em.offsets_of(lengths).to(DEV)
    t = sum(lengths)
    g = seeded(40)
    x, grad = em.small_integers((t, k), g, 1), em.small_integers((t, n), g, 1)
    w = em.small_integers((3, n, k), g, 1)

    def moved(v):
        whole = torch.zeros(v.numel() + 1, device=DEV, dtype=torch.bfloat16)
        whole[1:] = bf(v).flatten()
        return whole[1:].view(v.shape)

    want = torch.cat([x[a:z] @ w[e].t() for e, (a, z) in enumerate(groups(lengths))])
    want_dx = torch.cat([grad[a:z] @ w[e] for e, (a, z) in enumerate(groups(lengths))])
    want_dw = torch.stack([grad[a:z].t() @ x[a:z] for a, z in groups(lengths)])
    for fx in (bf, moved):
        for fw in (bf, moved):
            for fo in (bf, moved):
                y = grouped.gemm_grouped_bf16_into(fx(x), fw(w), off, fo(torch.zeros(t, n)))
                assert torch.equal(y.float().cpu(), want)
                dx = grouped.gemm_grouped_bf16_grad_input_into(fx(grad), fw(w), off,
                                                               fo(torch.zeros(t, k)))
                assert torch.equal(dx.float().cpu(), want_dx)
                dw = grouped.gemm_grouped_bf16_grad_weight_into(fx(grad), fw(x), off,
                                                                fo(torch.zeros(3, n, k)))
                assert torch.equal(dw.float().cpu(), want_dw)
    assert b.gemm_status() == 0


def test_offsets_past_32_bits():
    """Weights of more than 2**31 values, and the last expert's rows on them."""
    experts, n, k = 9, 16384, 14848
    assert experts * n * k > 2 ** 31
    w = torch.zeros(experts, n, k, device=DEV, dtype=torch.bfloat16)
    g = seeded(50)
    tail = em.small_integers((n, 48), g, 1)
    w[-1, :, -48:] = bf(tail)
    x = torch.zeros(200, k, device=DEV, dtype=torch.bfloat16)
    rows = em.small_integers((200, 48), g, 1)
    x[:, -48:] = bf(rows)
    off = em.offsets_of([0] * (experts - 1) + [200]).to(DEV)
    y = grouped.gemm_grouped_bf16(x, w, off)
    assert torch.equal(y.float().cpu(), rows @ tail.t())
    grad = torch.zeros(200, n, device=DEV, dtype=torch.bfloat16)
    grad[:, -1] = 1
    dx = grouped.gemm_grouped_bf16_grad_input(grad, w, off)
    assert torch.equal(dx[:, -48:].float().cpu(), tail[-1:].expand(200, -1))
    assert not dx[:, :-48].any()
    del w
    dw = grouped.gemm_grouped_bf16_grad_weight(grad, x, off)
    assert torch.equal(dw[-1, -1, -48:].float().cpu(), rows.sum(0))
    assert not dw[:-1].any() and not dw[-1, :-1].any()
    assert b.gemm_status() == 0


def test_outputs_past_32_bits():
    t, n, k = 140_000, 16384, 16
    assert t * n > 2 ** 31
    x = torch.zeros(t, k, device=DEV, dtype=torch.bfloat16)
    x[:, 0] = torch.arange(t, device=DEV) % 128
    w = torch.zeros(2, n, k, device=DEV, dtype=torch.bfloat16)
    w[0, :, 0], w[1, :, 0] = 1, 2
    off = em.offsets_of([1000, t - 1000]).to(DEV)
    y = grouped.gemm_grouped_bf16(x, w, off)
    want = x[:, 0].float() * torch.where(torch.arange(t, device=DEV) < 1000, 1.0, 2.0)
    for lo in range(0, t, 20_000):
        assert (y[lo:lo + 20_000].float() == want[lo:lo + 20_000, None]).all()
    assert b.gemm_status() == 0


def test_captured_layer_replays_with_other_offsets():
    """A whole layer (products, SwiGLU, both gradients) in a graph; the next
    replay reads other rows and other offsets.  An eager pass between the
    replays does not disturb it."""
    t, experts, n, k = 150, 4, 128, 64
    g = seeded(60)
    x = torch.randn(t, k, generator=g).bfloat16().to(DEV)
    up = torch.randn(experts, 2 * n, k, generator=g).mul(0.1).bfloat16().to(DEV)
    down = torch.randn(experts, k, n, generator=g).mul(0.1).bfloat16().to(DEV)
    off = em.offsets_of([100, 0, 20, 30]).to(DEV)

    def layer():
        h = grouped.gemm_grouped_swiglu_bf16(x, up, off)
        y = grouped.gemm_grouped_bf16(h, down, off)
        return (y, *grouped.gemm_grouped_bf16_backward(y, h, down, off))

    layer()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = layer()
    for lengths in ([0, 150, 0, 0], [1, 64, 65, 20]):
        off.copy_(em.offsets_of(lengths))
        x.copy_(torch.randn(t, k, generator=g).bfloat16())
        graph.replay()
        want = layer()
        torch.cuda.synchronize()
        for got, w in zip(captured, want):
            assert torch.equal(got, w)
    assert b.gemm_status() == 0
    del graph


def test_first_call_of_a_process_inside_a_capture():
    """Nothing that the library sets up on its first call breaks a capture."""
    code = """
import sys, torch
sys.path.insert(0, sys.argv[1])
from cuda_operator_lab import bindings, fp8, grouped
x = torch.ones(40, 256, device="cuda", dtype=torch.bfloat16)
w = torch.ones(2, 256, 256, device="cuda", dtype=torch.bfloat16)
off = torch.tensor([0, 30, 40], dtype=torch.int32, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = grouped.gemm_grouped_bf16(x, w, off)
    dx, dw = grouped.gemm_grouped_bf16_backward(y, x, w, off)
    y8 = grouped.gemm_grouped_fp8_block128(
        *fp8.quantize_fp8_block128(x), *fp8.quantize_fp8_block128_weight(w), off)
graph.replay()
torch.cuda.synchronize()
assert (y == 256).all() and (y8 == 256).all() and (dx == 65536).all()
assert (dw[0] == 7680).all() and (dw[1] == 2560).all()
assert bindings.gemm_status() == 0
print("captured")
"""
    done = subprocess.run([sys.executable, "-c", code, str(PACKAGE_DIR)], capture_output=True,
                          text=True, timeout=300)
    assert done.returncode == 0 and "captured" in done.stdout, done.stdout + done.stderr


def test_two_streams_at_once():
    """Two calls in flight on two streams share nothing."""
    lengths, n, k = [300, 0, 500, 41], 512, 1024
    off = em.offsets_of(lengths).to(DEV)
    g = seeded(70)
    xs = [torch.randn(sum(lengths), k, generator=g).bfloat16().to(DEV) for _ in range(2)]
    w = torch.randn(4, n, k, generator=g).bfloat16().to(DEV)
    want = [grouped.gemm_grouped_bf16(x, w, off) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(grouped.gemm_grouped_bf16(xs[i], w, off))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])
    assert b.gemm_status() == 0


def test_results_repeat_bit_for_bit():
    lengths, n, k = [300, 0, 500, 41], 520, 1032
    off = em.offsets_of(lengths).to(DEV)
    g = seeded(80)
    x = torch.randn(sum(lengths), k, generator=g).bfloat16().to(DEV)
    w = torch.randn(4, n, k, generator=g).bfloat16().to(DEV)
    grad = torch.randn(sum(lengths), n, generator=g).bfloat16().to(DEV)
    first = (grouped.gemm_grouped_bf16(x, w, off),
             *grouped.gemm_grouped_bf16_backward(grad, x, w, off))
    for _ in range(3):
        again = (grouped.gemm_grouped_bf16(x, w, off),
                 *grouped.gemm_grouped_bf16_backward(grad, x, w, off))
        assert all(torch.equal(p, q) for p, q in zip(first, again))


# ---------------------------------------------------------------- together


def test_expert_layer_in_8_bits_beside_bf16():
    """One MLP layer of experts as a server runs it: rows sorted by expert,
    quantise, gate/up with SwiGLU, quantise, down; and the same in bf16.  Each
    step is held to the bound of its own operands; the two layers differ by the
    quantisation."""
    experts, t, k, n = 6, 90, 512, 256
    g = seeded(90)
    tokens = torch.randn(t, k, generator=g).bfloat16()
    choice = torch.randint(0, experts, (t,), generator=g)
    choice[choice == 2] = 3  # an expert without rows
    order = torch.argsort(choice, stable=True)
    off = em.offsets_of(torch.bincount(choice, minlength=experts).tolist()).to(DEV)
    up = (torch.randn(experts, 2 * n, k, generator=g) * k ** -0.5).bfloat16().to(DEV)
    down = (torch.randn(experts, k, n, generator=g) * n ** -0.5).bfloat16().to(DEV)
    x = tokens[order].to(DEV)

    h = grouped.gemm_grouped_swiglu_bf16(x, up, off)
    y = grouped.gemm_grouped_bf16(h, down, off)

    upq, downq = fp8.quantize_fp8_block128_weight(up), fp8.quantize_fp8_block128_weight(down)
    xq = fp8.quantize_fp8_block128(x)
    h8 = grouped.gemm_grouped_swiglu_fp8_block128(*xq, *upq, off)
    hq = fp8.quantize_fp8_block128(h8)
    y8 = grouped.gemm_grouped_fp8_block128(*hq, *downq, off)
    assert b.gemm_status() == 0

    def back(pair, height):
        return pair[0].double() * em.spread(pair[1], height, *pair[0].shape[-2:])

    ends = off.tolist()
    for e, (lo, hi) in enumerate(zip(ends[:-1], ends[1:])):
        em.assert_within(h[lo:hi], *em.product(x[lo:hi].double(), up[e].double(), True))
        em.assert_within(y[lo:hi], *em.product(h[lo:hi].double(), down[e].double(), False))
        em.assert_within(h8[lo:hi], *em.product(back(xq, 1)[lo:hi], back(upq, 128)[e], True))
        em.assert_within(y8[lo:hi], *em.product(back(hq, 1)[lo:hi], back(downq, 128)[e], False))
    # e4m3 keeps 3 bits behind the leading one: each operand is off by at most
    # 2**-4 of its value, four quantised operands in two products
    err = (y8.double() - y.double()).norm() / y.double().norm()
    assert err < 4 * 2.0 ** -4
    # a dense call is the grouped one with a single expert
    one = torch.tensor([0, t], dtype=torch.int32, device=DEV)
    dense = fp8.gemm_swiglu_fp8_block128(*xq, upq[0][0], upq[1][0])
    single = grouped.gemm_grouped_swiglu_fp8_block128(*xq, upq[0][:1], upq[1][:1], one)
    assert torch.allclose(dense.float(), single.float(), rtol=2.0 ** -7, atol=1e-6)
