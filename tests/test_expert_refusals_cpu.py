"""What the expert-layer operators refuse, checked without a GPU (CPU).

Arguments are checked before the device, so every refusal shows on CPU tensors;
a call that is right in all but its device names CUDA.
"""

from __future__ import annotations

import pytest
import torch

from cuda_operator_lab import bindings, fp8, grouped
from expert_math import offsets_of

E4M3 = torch.float8_e4m3fn


def bf(*shape):
    return torch.zeros(shape, dtype=torch.bfloat16)


def f32(*shape):
    return torch.zeros(shape, dtype=torch.float32)


def f8(*shape):
    return torch.zeros(shape, dtype=torch.float32).to(E4M3)


OFFSETS = offsets_of([2, 0, 3])

GOOD = {
    "quantize_fp8_block128_into": [bf(3, 200), f8(3, 200), f32(3, 2)],
    "quantize_fp8_block128": [f32(3, 200)],
    "quantize_fp8_block128_weight_into": [f32(2, 130, 200), f8(2, 130, 200), f32(2, 2, 2)],
    "quantize_fp8_block128_weight": [bf(130, 200)],
    "gemm_fp8_block128_into": [f8(3, 200), f32(3, 2), f8(130, 200), f32(2, 2), bf(3, 130)],
    "gemm_fp8_block128": [f8(3, 200), f32(3, 2), f8(130, 200), f32(2, 2)],
    "gemm_swiglu_fp8_block128_into": [f8(3, 200), f32(3, 2), f8(256, 200), f32(2, 2), bf(3, 128)],
    "gemm_swiglu_fp8_block128": [f8(3, 200), f32(3, 2), f8(256, 200), f32(2, 2)],
    "gemm_grouped_bf16_into": [bf(5, 24), bf(3, 10, 24), OFFSETS, bf(5, 10)],
    "gemm_grouped_bf16": [bf(5, 24), bf(3, 10, 24), OFFSETS],
    "gemm_grouped_swiglu_bf16_into": [bf(5, 24), bf(3, 10, 24), OFFSETS, bf(5, 5)],
    "gemm_grouped_swiglu_bf16": [bf(5, 24), bf(3, 10, 24), OFFSETS],
    "gemm_grouped_bf16_grad_input_into": [bf(5, 10), bf(3, 10, 24), OFFSETS, bf(5, 24)],
    "gemm_grouped_bf16_grad_input": [bf(5, 10), bf(3, 10, 24), OFFSETS],
    "gemm_grouped_bf16_grad_weight_into": [bf(5, 10), bf(5, 24), OFFSETS, bf(3, 10, 24)],
    "gemm_grouped_bf16_grad_weight": [bf(5, 10), bf(5, 24), OFFSETS],
    "gemm_grouped_bf16_backward": [bf(5, 10), bf(5, 24), bf(3, 10, 24), OFFSETS],
    "gemm_grouped_fp8_block128_into": [f8(5, 200), f32(5, 2), f8(3, 130, 200), f32(3, 2, 2),
                                       OFFSETS, bf(5, 130)],
    "gemm_grouped_fp8_block128": [f8(5, 200), f32(5, 2), f8(3, 130, 200), f32(3, 2, 2), OFFSETS],
    "gemm_grouped_swiglu_fp8_block128_into": [f8(5, 200), f32(5, 2), f8(3, 256, 200),
                                              f32(3, 2, 2), OFFSETS, bf(5, 128)],
    "gemm_grouped_swiglu_fp8_block128": [f8(5, 200), f32(5, 2), f8(3, 256, 200), f32(3, 2, 2),
                                         OFFSETS],
}


def operator(name):
    return getattr(fp8 if hasattr(fp8, name) else grouped, name)


def refused(name, args, error=ValueError, match=None):
    """The call is refused for its arguments, not for being on the CPU."""
    with pytest.raises(error, match=match) as info:
        operator(name)(*args)
    assert "CUDA" not in str(info.value), (name, str(info.value))


def test_every_public_operator_is_covered():
    assert set(GOOD) == set(fp8.__all__) | set(grouped.__all__)


@pytest.mark.parametrize("name", sorted(GOOD))
def test_cpu_tensors_are_refused(name):
    with pytest.raises(ValueError, match="CUDA"):
        operator(name)(*GOOD[name])


@pytest.mark.parametrize("name", sorted(GOOD))
def test_each_argument_of_another_type_is_refused(name):
    for i, arg in enumerate(GOOD[name]):
        args = list(GOOD[name])
        args[i] = arg.double()
        refused(name, args, TypeError)


@pytest.mark.parametrize("name", sorted(GOOD))
def test_each_argument_of_another_rank_is_refused(name):
    for i, arg in enumerate(GOOD[name]):
        args = list(GOOD[name])
        args[i] = arg[None, None]
        refused(name, args)


@pytest.mark.parametrize("name", sorted(GOOD))
def test_each_argument_of_another_shape_is_refused(name):
    # (argument, dimension) whose length nothing else fixes
    free = {
        "quantize_fp8_block128": {(0, 0), (0, 1)},
        "quantize_fp8_block128_weight": {(0, 0), (0, 1)},
        "gemm_fp8_block128": {(2, 0)},
        "gemm_grouped_fp8_block128": {(2, 1)},
        "gemm_grouped_bf16": {(0, 0), (1, 1)},
        "gemm_grouped_swiglu_bf16": {(0, 0)},
        "gemm_grouped_bf16_grad_input": {(0, 0), (1, 2)},
        "gemm_grouped_bf16_grad_weight": {(0, 1), (1, 1), (2, 0)},
    }.get(name, set())
    for i, arg in enumerate(GOOD[name]):
        for dim in range(arg.ndim):
            if (i, dim) in free:
                continue
            args = list(GOOD[name])
            longer = torch.cat([arg.float(), arg.float().narrow(dim, 0, 1)], dim)
            args[i] = longer.to(arg.dtype)
            refused(name, args)


@pytest.mark.parametrize("name", sorted(GOOD))
def test_each_argument_with_strides_is_refused(name):
    for i, arg in enumerate(GOOD[name]):
        args = list(GOOD[name])
        args[i] = torch.stack([arg.float(), arg.float()], -1).to(arg.dtype)[..., 0]
        assert not args[i].is_contiguous() and args[i].shape == arg.shape
        with pytest.raises(ValueError, match="contiguous"):
            operator(name)(*args)


def test_swiglu_needs_whole_gate_and_up_rows():
    with pytest.raises(ValueError, match="even"):
        grouped.gemm_grouped_swiglu_bf16(bf(5, 24), bf(3, 9, 24), OFFSETS)
    for rows in (130, 384):  # gate rows end inside a tile of scales
        blocks = -(-rows // 128)
        with pytest.raises(ValueError, match="whole blocks"):
            fp8.gemm_swiglu_fp8_block128(f8(3, 200), f32(3, 2), f8(rows, 200), f32(blocks, 2))
        with pytest.raises(ValueError, match="whole blocks"):
            grouped.gemm_grouped_swiglu_fp8_block128(f8(5, 200), f32(5, 2), f8(3, rows, 200),
                                                     f32(3, blocks, 2), OFFSETS)


def test_products_over_nothing_are_refused():
    with pytest.raises(ValueError, match="k > 0"):
        fp8.gemm_fp8_block128(f8(3, 0), f32(3, 0), f8(8, 0), f32(1, 0))
    with pytest.raises(ValueError, match="k > 0"):
        grouped.gemm_grouped_bf16(bf(5, 0), bf(3, 8, 0), OFFSETS)
    with pytest.raises(ValueError, match="n > 0"):
        grouped.gemm_grouped_bf16_grad_input(bf(5, 0), bf(3, 0, 8), OFFSETS)


def test_too_many_experts_are_refused():
    many = grouped.MAX_EXPERTS + 1
    with pytest.raises(ValueError, match="at most"):
        grouped.gemm_grouped_bf16(bf(5, 8), bf(many, 8, 8), offsets_of([0] * many))
    with pytest.raises(ValueError, match="at most"):
        grouped.gemm_grouped_bf16_grad_weight(bf(5, 8), bf(5, 8), offsets_of([0] * many))


def test_sizes_past_the_limit_are_refused():
    big = torch.empty(1, dtype=torch.bfloat16).expand(2 ** 31, 8)  # no memory behind it
    with pytest.raises(ValueError, match="at most"):
        fp8.quantize_fp8_block128_into(big, torch.empty(1).to(E4M3).expand(2 ** 31, 8),
                                       torch.empty(1).expand(2 ** 31, 1))


def library():
    from test_abi import library as build

    build()
    return bindings._library().handle


def test_c_entries_refuse_bad_sizes_and_pointers():
    """The C entries check before any launch: no device is needed to be refused."""
    lib = library()
    invalid = 1
    p = 1 << 20  # a pointer that is never used
    call = {
        "quantize": lambda x, q, s, m, k: lib.cuda_operator_quantize_fp8_block128_bf16(x, q, s, m, k, None),
        "tiles": lambda x, q, s, e, n, k: lib.cuda_operator_quantize_fp8_block128_weight_f32(x, q, s, e, n, k, None),
        "fp8": lambda *a: lib.cuda_operator_gemm_fp8_block128(*a, None),
        "fp8s": lambda *a: lib.cuda_operator_gemm_swiglu_fp8_block128(*a, None),
        "g": lambda *a: lib.cuda_operator_gemm_grouped_bf16(*a, None),
        "gs": lambda *a: lib.cuda_operator_gemm_grouped_swiglu_bf16(*a, None),
        "g8": lambda *a: lib.cuda_operator_gemm_grouped_fp8_block128(*a, None),
        "g8s": lambda *a: lib.cuda_operator_gemm_grouped_swiglu_fp8_block128(*a, None),
        "dx": lambda *a: lib.cuda_operator_gemm_grouped_bf16_grad_input(*a, None),
        "dw": lambda *a: lib.cuda_operator_gemm_grouped_bf16_grad_weight(*a, None),
    }
    call["both"] = lambda *a: lib.cuda_operator_gemm_grouped_bf16_backward(*a, None)
    for null in range(6):
        args = [p] * 6
        args[null] = None
        assert call["both"](*args, 4, 8, 8, 2) == invalid, null
    assert call["both"](*[p] * 6, 1 << 31, 8, 8, 2) == invalid
    assert call["both"](*[p] * 6, 4, 8, 8, 1025) == invalid
    assert call["both"](*[None] * 6, 0, 0, 8, 2) == 0
    # nothing to do succeeds before any check
    assert call["quantize"](None, None, None, 0, 8) == 0
    assert call["tiles"](None, None, None, 0, 8, 8) == 0
    assert call["fp8"](None, None, None, None, None, 0, 8, 8) == 0
    assert call["g"](None, None, None, None, 0, 8, 8, 2) == 0
    assert call["g8"](None, None, None, None, None, None, 4, 8, 8, 0) == 0
    assert call["dx"](None, None, None, None, 0, 8, 8, 2) == 0
    assert call["dw"](None, None, None, None, 4, 8, 0, 2) == 0
    for null in range(3):
        args = [p, p, p]
        args[null] = None
        assert call["quantize"](*args, 4, 8) == invalid
        assert call["tiles"](*args, 2, 4, 8) == invalid
    for null in range(5):
        args = [p] * 5
        args[null] = None
        assert call["fp8"](*args, 4, 8, 8) == invalid
        assert call["fp8s"](*args, 4, 8, 128) == invalid
    for null in range(6):
        args = [p] * 6
        args[null] = None
        assert call["g8"](*args, 4, 8, 8, 2) == invalid
        assert call["g8s"](*args, 4, 8, 128, 2) == invalid
    for null in range(4):
        args = [p] * 4
        args[null] = None
        for name in ("g", "gs", "dx", "dw"):
            assert call[name](*args, 4, 8, 8, 2) == invalid, (name, null)
    huge = 1 << 31
    for sizes in ((huge, 8, 8, 2), (4, huge, 8, 2), (4, 8, huge, 2), (4, 8, 8, 1025)):
        for name in ("g", "gs", "dx", "dw"):
            assert call[name](*[p] * 4, *sizes) == invalid, (name, sizes)
        assert call["g8"](*[p] * 6, *sizes) == invalid
    for name in ("g", "gs"):  # no columns to sum over
        assert call[name](*[p] * 4, 4, 0, 8, 2) == invalid
    assert call["dx"](*[p] * 4, 4, 8, 0, 2) == invalid
    assert call["fp8"](*[p] * 5, 4, 0, 8) == invalid
    assert call["fp8s"](*[p] * 5, 4, 8, 100) == invalid  # gate rows end inside a tile
    assert call["quantize"](p, p, p, huge, 8) == invalid
    assert call["tiles"](p, p, p, huge, 8, 8) == invalid
