"""Block-scaled e4m3 products whose two scales multiply out of fp32's normal range (GPU).

A scale is any fp32 number, so the product of a row's and a tile's may overflow
or lose its bits to a subnormal where the scaled sum itself is an ordinary
number.  Results are held to 64-bit forms under the bounds of expert_math; bf16
rounds results below 2**-126 to multiples of 2**-133, half of which is added.
"""

from __future__ import annotations

import pytest
import torch

import expert_math as em
from conftest import seeded
from cuda_operator_lab import bindings as b
from cuda_operator_lab import fp8, grouped

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3 = torch.float8_e4m3fn

# rows, columns, K: sums shared by clusters, single CTAs of 128 and 256 columns,
# CTA pairs, and rows that TMA cannot address (K % 16 != 0)
SHAPES = [(3, 256, 4096), (40, 128, 1040), (300, 640, 1040), (700, 2048, 528), (2100, 4096, 400),
          (70, 256, 1000)]


def near(v, g):
    """Scales around v: a random factor in [1, 2)."""
    return lambda *shape: (v * (1 + torch.rand(*shape, generator=g))).float()


def values(shape, g, low, high):
    """e4m3 values of one sign between two powers of two."""
    return torch.exp2(torch.empty(shape).uniform_(low, high, generator=g)).clamp(max=448).to(E4M3)


def run(x, xs, w, ws, swiglu, by_expert):
    x, xs, w, ws = (v.to(DEV) for v in (x, xs, w, ws))
    if by_expert:
        off = torch.tensor([0, x.shape[0]], dtype=torch.int32, device=DEV)
        gemm = grouped.gemm_grouped_swiglu_fp8_block128 if swiglu else grouped.gemm_grouped_fp8_block128
        y = gemm(x, xs, w[None], ws[None], off)
    else:
        y = (fp8.gemm_swiglu_fp8_block128 if swiglu else fp8.gemm_fp8_block128)(x, xs, w, ws)
    assert b.gemm_status() == 0
    xd = x.double() * em.spread(xs, 1, *x.shape)
    wd = w.double() * em.spread(ws, 128, *w.shape)
    want, bound = em.product(xd, wd, swiglu)
    assert (want.abs().amax() > 0) and torch.isfinite(want).all()
    y = y.double()
    assert torch.isfinite(y).all()
    excess = (y - want).abs() - bound - 2.0 ** -134
    assert float(excess.max()) <= 0, f"off by {float(excess.max())} more than the bound"
    return y


@pytest.mark.parametrize("by_expert", [False, True])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_products_of_tiny_scales(m, n, k, by_expert):
    """2**-112 times 2**-36 is a subnormal of one or two bits; the blocks' sums of
    values near 448 bring the result back above 2**-126."""
    g = seeded(m)
    kb = -(-k // 128)
    x, w = values((m, k), g, 8, 8.8), values((n, k), g, 8, 8.8)
    run(x, near(2.0 ** -112, g)(m, kb), w, near(2.0 ** -36, g)(-(-n // 128), kb), False, by_expert)


@pytest.mark.parametrize("by_expert", [False, True])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_products_of_huge_scales(m, n, k, by_expert):
    """2**83 times 2**48 is past fp32's range; sums of zero stay zero and small sums
    stay finite.  Signs alternate from row to row of w."""
    g = seeded(m + 1)
    kb = -(-k // 128)
    x, w = values((m, k), g, -9, -7).float(), values((n, k), g, -9, -7).float()
    x[:, ::3] = 0
    w[:, 1::3] = 0
    x[torch.rand(m, k, generator=g) < 0.9] = 0
    w[::2] *= -1
    run(x.to(E4M3), near(2.0 ** 83, g)(m, kb), w.to(E4M3), near(2.0 ** 48, g)(-(-n // 128), kb),
        False, by_expert)


@pytest.mark.parametrize("by_expert", [False, True])
@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("up_scale", [-36, 45])
def test_swiglu_of_extreme_up_scales(m, n, k, up_scale, by_expert):
    """The gate's scales multiply to ordinary numbers, the up rows' do not."""
    n //= 2
    n = -(-n // 128) * 128
    g = seeded(m + 2)
    kb = -(-k // 128)
    x = values((m, k), g, -9, -7) if up_scale > 0 else values((m, k), g, 8, 8.8)
    w = torch.cat([values((n, k), g, -9, -7), x.new_zeros(n, k).to(E4M3)])
    w[n:] = values((n, k), g, -9, -7) if up_scale > 0 else values((n, k), g, 8, 8.8)
    x_exp = 83 if up_scale > 0 else -112
    xs = near(2.0 ** x_exp, g)(m, kb)
    # gate sums of order one
    gate = float((x.double().mean() * w[:n].double().mean() * k).log2().round())
    gate_scale = near(2.0 ** (-x_exp - gate - 1), g)(n // 128, kb)
    up = near(2.0 ** up_scale, g)(n // 128, kb)
    run(x, xs, w, torch.cat([gate_scale, up]), True, by_expert)


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_rows_of_extreme_scales_change_no_other(m, n, k):
    """Every second row's scales are extreme, zero or negative: the others' results
    are those of a call without such rows, bit for bit."""
    g = seeded(m + 3)
    kb, nb = -(-k // 128), -(-n // 128)
    x, w = torch.randn(m, k, generator=g).to(E4M3), torch.randn(n, k, generator=g).to(E4M3)
    xs, ws = near(0.25, g)(m, kb), near(2.0 ** -20, g)(nb, kb)
    plain = run(x, xs, w, ws, False, False)
    odd = xs.clone()
    for i, v in enumerate((2.0 ** -120, 0.0, -3.0, 2.0 ** 126, 2.0 ** -149)):
        odd[1 + 2 * i::10] = v
    y = fp8.gemm_fp8_block128(x.to(DEV), odd.to(DEV), w.to(DEV), ws.to(DEV)).double()
    assert b.gemm_status() == 0
    assert torch.equal(y[::2], plain[::2])
    assert torch.isfinite(y).all()
    assert (y[3::10] == 0).all()
    # a zero scale beside a huge one
    y = fp8.gemm_fp8_block128(x.to(DEV), torch.zeros_like(xs).to(DEV), w.to(DEV),
                              torch.full_like(ws, 2.0 ** 126).to(DEV))
    assert (y == 0).all()
