"""e4m3 block-128 quantiser and products against 64-bit forms (GPU).

Tolerances are those of expert_math (derived there); quantised values are those
of the exact quotient, ties to even.
"""

from __future__ import annotations

import pytest
import torch

import expert_math as em
from conftest import seeded
from cuda_operator_lab import bindings as b
from cuda_operator_lab import fp8

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3 = torch.float8_e4m3fn


def check_quantized(x: torch.Tensor, q: torch.Tensor, scale: torch.Tensor, height: int) -> None:
    """One matrix: values and scales against 64 bits."""
    before, want_scale = em.quantize(x.cpu(), height)
    # one division: half a step of fp32
    assert ((scale.cpu().double() - want_scale).abs() <= 2.0 ** -24 * want_scale).all()
    got = q.cpu().double()
    assert torch.equal(got, em.grid_e4m3(before))


SHAPES = [(1, 1), (1, 128), (1, 4096), (3, 127), (5, 129), (7, 1000), (33, 264), (200, 2064),
          (1, 16), (129, 136), (5000, 512), (5003, 520)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_rows(shape, dtype):
    x = (torch.randn(shape, generator=seeded(1)) * torch.rand(shape[1], generator=seeded(2)) * 9).to(dtype)
    q, scale = fp8.quantize_fp8_block128(x.to(DEV))
    assert q.dtype == E4M3 and q.shape == x.shape
    check_quantized(x, q, scale, 1)


@pytest.mark.parametrize("shape", [(1, 1, 1), (2, 128, 128), (3, 130, 200), (1, 127, 129),
                                   (2, 1, 4096), (4, 300, 520), (2, 77, 75)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_weights(shape, dtype):
    w = torch.randn(shape, generator=seeded(3)).to(dtype)
    q, scale = fp8.quantize_fp8_block128_weight(w.to(DEV))
    for e in range(shape[0]):
        check_quantized(w[e], q[e], scale[e], 128)
    one, one_scale = fp8.quantize_fp8_block128_weight(w[0].to(DEV))
    assert torch.equal(one.float(), q[0].float()) and torch.equal(one_scale, scale[0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("exponent", [0, -90, 100, -99])
def test_quantize_ties(dtype, exponent):
    """Quotients that are ties between e4m3 values, or next to one, at every step
    of its range, subnormal steps included: the largest of a row fixes 448 / a."""
    g = seeded(5)
    steps = torch.arange(0, 2 ** 4 * 16).double()
    ties = torch.cat([(2 * steps + 1) * 2.0 ** -10, (2 * torch.arange(8, 16).repeat(14) + 1).double()
                      * 2.0 ** torch.arange(-10, 4).repeat_interleave(8).double()])
    ties = ties[ties < 448]
    rows = []
    for top in (448.0, 1.0, 7.0, 1.75, 1.171875, 3.140625, float(torch.rand(1, generator=g) + 1)):
        x = (ties * top / 448).float()
        for nudge in (0, 1, -1, 2, -2):  # units in the last place of the source type
            near = x.to(dtype).view(torch.int16 if dtype == torch.bfloat16 else torch.int32) + nudge
            near = near.view(dtype).float().clamp(-top, top)
            near = torch.nn.functional.pad(near, (0, -near.numel() % 127)).view(-1, 127)
            sign = torch.randint(0, 2, near.shape, generator=g) * 2 - 1
            rows.append(torch.cat([torch.full((near.shape[0], 1), top), near * sign], 1))
    x = (torch.cat(rows) * 2.0 ** exponent).to(dtype)
    q, scale = fp8.quantize_fp8_block128(x.to(DEV))
    check_quantized(x, q, scale, 1)
    w = x[: x.shape[0] // 128 * 128]
    q, scale = fp8.quantize_fp8_block128_weight(w.to(DEV))
    check_quantized(w, q, scale, 128)


@pytest.mark.parametrize("offset", [1, 2, 3])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_unaligned_base(offset, dtype):
    """Views that start off a 16-byte boundary, and outputs off an 8-byte one."""
    x = torch.randn(6 * 256 + offset, generator=seeded(4)).to(dtype).to(DEV)[offset:].view(6, 256)
    q = torch.zeros(6 * 256 + offset, device=DEV, dtype=torch.uint8)[offset:].view(E4M3).view(6, 256)
    scale = torch.empty(6, 2, device=DEV)
    assert fp8.quantize_fp8_block128_into(x, q, scale)[0] is q
    check_quantized(x, q, scale, 1)
    tiles = torch.empty(1, 2, device=DEV)
    fp8.quantize_fp8_block128_weight_into(x, q, tiles)
    check_quantized(x, q, tiles, 128)


def test_quantize_extreme_values():
    """All-zero and tiny blocks, the largest values, NaN and infinities."""
    x = torch.zeros(8, 256)
    x[1] = 2.0 ** -120                       # under the floor: rounds to zero
    x[2, :128] = 3.0e38
    x[2, 5] = -3.3e38
    x[3, 130] = float("nan")
    x[4, 3] = float("inf")
    x[4, 4] = 1.0
    x[5, 200] = float("-inf")
    x[6] = torch.arange(256) * 2.0 ** -126   # subnormals and just above
    x[7] = 1e-30
    q, scale = (t.cpu() for t in fp8.quantize_fp8_block128(x.to(DEV)))
    v = q.float()
    floor = torch.tensor(2.0 ** -100) / 448
    assert (v[0] == 0).all() and (scale[0] == floor).all()
    assert (v[1] == 0).all() and (scale[1] == floor).all()
    check_quantized(x[2:3], q[2:3], scale[2:3], 1)
    assert torch.isnan(scale[3, 1]) and torch.isnan(v[3, 128:]).all() and (v[3, :128] == 0).all()
    assert torch.isinf(scale[4, 0]) and torch.isnan(v[4, 3]) and v[4, 4] == 0
    assert torch.isinf(scale[5, 1]) and torch.isnan(v[5, 200]) and (v[5, 128:200] == 0).all()
    check_quantized(x[6:], q[6:], scale[6:], 1)
    # a product over such a block is NaN, over the other rows it is not
    w = torch.ones(64, 256).to(E4M3).to(DEV)
    y = fp8.gemm_fp8_block128(q.to(DEV), scale.to(DEV), w, torch.ones(1, 2, device=DEV))
    assert torch.isnan(y[[3, 4, 5]]).all()
    assert torch.isfinite(y[[0, 1, 6, 7]]).all()


def operands(m, n, k, g, swiglu=False):
    x = torch.randn(m, k, generator=g) * torch.exp(torch.randn(k, generator=g))
    w = torch.randn(2 * n if swiglu else n, k, generator=g) * k ** -0.5
    xq, xs = fp8.quantize_fp8_block128(x.to(DEV))
    wq, ws = fp8.quantize_fp8_block128_weight(w.to(DEV))
    return xq, xs, wq, ws


def dequantized(xq, xs, wq, ws):
    return (xq.double() * em.spread(xs, 1, *xq.shape), wq.double() * em.spread(ws, 128, *wq.shape))


# one token to several tiles; k of one block, partial blocks, many blocks; odd n
PRODUCTS = [(1, 128, 128), (1, 4096, 4096), (2, 16, 16), (7, 129, 144), (16, 1000, 1040),
            (17, 264, 4112), (64, 512, 272), (127, 255, 400), (128, 256, 512), (129, 257, 528),
            (300, 1001, 2064), (256, 320, 1024), (513, 384, 640), (1025, 640, 896),
            # sums shared by the CTAs of a cluster, 64 and 128 columns a tile
            (3, 200, 14336), (32, 4096, 1040), (33, 600, 2064), (40, 2900, 1040), (96, 1000, 784),
            (5, 4100, 4096)]


@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_gemm(m, n, k):
    args = operands(m, n, k, seeded(m + n + k))
    y = fp8.gemm_fp8_block128(*args)
    assert y.shape == (m, n) and y.dtype == torch.bfloat16
    assert b.gemm_status() == 0
    em.assert_within(y, *em.product(*dequantized(*args), False))


@pytest.mark.parametrize("m,n,k", [(1, 128, 128), (1, 2048, 4096), (5, 256, 400), (130, 384, 1040),
                                   (257, 128, 2064), (600, 640, 528), (2, 256, 8208),
                                   (31, 1024, 1040), (70, 512, 2064)])
def test_gemm_swiglu(m, n, k):
    args = operands(m, n, k, seeded(m + n + k), swiglu=True)
    y = fp8.gemm_swiglu_fp8_block128(*args)
    assert y.shape == (m, n)
    assert b.gemm_status() == 0
    em.assert_within(y, *em.product(*dequantized(*args), True))


@pytest.mark.parametrize("m,n,k", [(1, 130, 64), (40, 300, 100), (130, 100, 37), (300, 200, 1)])
def test_gemm_of_small_integers_is_exact(m, n, k):
    """Sums of at most 256 in steps of one, and any K: rows TMA cannot address too."""
    g = seeded(k)
    x, w = em.small_integers((m, k), g, 1), em.small_integers((n, k), g, 1)
    ones = torch.ones(m, 1, device=DEV)
    y = fp8.gemm_fp8_block128(x.to(E4M3).to(DEV), ones, w.to(E4M3).to(DEV),
                              torch.ones(-(-n // 128), 1, device=DEV))
    assert torch.equal(y.float().cpu(), x @ w.t())


def test_gemm_unaligned_operands():
    """x and w one byte off a 16-byte boundary; the output two bytes off."""
    g = seeded(8)
    m, n, k = 70, 90, 256
    xq, xs, wq, ws = operands(m, n, k, g)

    def moved(t):
        flat = torch.zeros(t.numel() + 1, device=DEV, dtype=torch.uint8)
        flat[1:] = t.view(torch.uint8).flatten()
        return flat[1:].view(E4M3).view(t.shape)

    want, bound = em.product(*dequantized(xq, xs, wq, ws), False)
    em.assert_within(fp8.gemm_fp8_block128(moved(xq), xs, wq, ws), want, bound)
    em.assert_within(fp8.gemm_fp8_block128(xq, xs, moved(wq), ws), want, bound)
    out = torch.zeros(m * n + 1, device=DEV, dtype=torch.bfloat16)[1:].view(m, n)
    em.assert_within(fp8.gemm_fp8_block128_into(xq, xs, wq, ws, out), want, bound)
    assert b.gemm_status() == 0


def test_rows_do_not_meet():
    """A NaN row of x and a NaN row of w spoil their own row and column alone."""
    m, n, k = 140, 200, 512
    xq, xs, wq, ws = operands(m, n, k, seeded(9))
    clean = fp8.gemm_fp8_block128(xq, xs, wq, ws)
    xq.view(torch.uint8)[131] = 0x7F
    wq.view(torch.uint8)[77] = 0x7F
    y = fp8.gemm_fp8_block128(xq, xs, wq, ws)
    assert torch.isnan(y[131]).all() and torch.isnan(y[:, 77]).all()
    rows = [i for i in range(m) if i != 131]
    cols = [j for j in range(n) if j != 77]
    assert torch.equal(y[rows][:, cols], clean[rows][:, cols])


def test_empty_calls():
    none = torch.empty(0, 256, device=DEV).to(E4M3)
    w, ws = fp8.quantize_fp8_block128_weight(torch.randn(64, 256, device=DEV))
    assert fp8.gemm_fp8_block128(none, torch.empty(0, 2, device=DEV), w, ws).shape == (0, 64)
    q, s = fp8.quantize_fp8_block128(torch.empty(0, 256, device=DEV))
    assert q.shape == (0, 256) and s.shape == (0, 2)
    q, s = fp8.quantize_fp8_block128_weight(torch.empty(0, 64, 256, device=DEV))
    assert q.shape == (0, 64, 256) and s.shape == (0, 1, 2)


def test_capture_and_another_stream():
    """A captured chain replays on new inputs; a call on a side stream is ordered by it."""
    g = seeded(10)
    x = torch.randn(50, 512, generator=g).to(DEV)
    wq, ws = fp8.quantize_fp8_block128_weight(torch.randn(512, 512, generator=g).to(DEV))
    fp8.gemm_swiglu_fp8_block128(*fp8.quantize_fp8_block128(x), wq, ws)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = fp8.gemm_swiglu_fp8_block128(*fp8.quantize_fp8_block128(x), wq, ws)
    for seed in (11, 12):
        x.copy_(torch.randn(50, 512, generator=seeded(seed)))
        graph.replay()
        want = fp8.gemm_swiglu_fp8_block128(*fp8.quantize_fp8_block128(x), wq, ws)
        torch.cuda.synchronize()
        assert torch.equal(y, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = fp8.gemm_swiglu_fp8_block128(*fp8.quantize_fp8_block128(x), wq, ws)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(again, want)
    assert b.gemm_status() == 0
    del graph


def test_results_repeat_bit_for_bit():
    for m in (1, 40, 700):
        args = operands(m, 1024, 2048, seeded(m))
        first = fp8.gemm_fp8_block128(*args)
        for _ in range(3):
            assert torch.equal(fp8.gemm_fp8_block128(*args), first)
