"""8-bit (e4m3) operands with a scale for each block of 128, and their products.

A matrix is held as ``torch.float8_e4m3fn`` values beside fp32 scales: one for
each 128 columns of a row (activations, ``[M, ceil(K/128)]``) or for each
128 x 128 tile (weights, ``[N/128, K/128]`` rounded up, with the experts in
front where there are several).  For a block with largest magnitude ``a`` (at
least 2**-100) the scale is ``a / 448`` and the values are ``x * 448 / a`` rounded
to nearest even (of the exact quotient), so ``q.float() * scale`` stands for
``x``.  A NaN or
an infinity in a block makes every product over that block NaN.  The products
take any finite fp32 scales, also ones whose product overflows or underflows
where the scaled sum does not.

As in ``bindings``: contiguous CUDA tensors, the current stream of the
operands' device, ``_into`` forms that return the caller's storage, no
synchronisation and no autograd.  The products take every K; they run on the
tensor cores where K is a multiple of 16 and the operands start on 16-byte
boundaries, elsewhere on a much slower CUDA-core kernel.
"""

from __future__ import annotations

import torch

from . import bindings
from .bindings import _ptr, _stream

try:
    from torch._C import _cuda_getDevice as _current_device
except ImportError:  # a torch without CUDA: every call is refused for its tensors
    from torch.cuda import current_device as _current_device

__all__ = [
    "quantize_fp8_block128", "quantize_fp8_block128_into",
    "quantize_fp8_block128_weight", "quantize_fp8_block128_weight_into",
    "gemm_fp8_block128", "gemm_fp8_block128_into",
    "gemm_swiglu_fp8_block128", "gemm_swiglu_fp8_block128_into",
]

BLOCK = 128
_E4M3 = torch.float8_e4m3fn
_MAX_SIZE = 0x7FFFFFFF - 1024


def _blocks(size: int) -> int:
    return -(-size // BLOCK)


def _placed(*tensors: torch.Tensor) -> bool:
    """Whether all are contiguous CUDA tensors of one device."""
    device = tensors[0].get_device()  # -1 off the GPU
    if device < 0:
        return False
    for t in tensors:
        if not t.is_contiguous() or t.get_device() != device:
            return False
    return True


def _check_placement(what: str, *tensors: torch.Tensor) -> None:
    if _placed(*tensors):
        return
    for t in tensors:
        if not t.is_contiguous():
            raise ValueError(f"all {what} tensors must be contiguous")
    for t in tensors:
        if not t.is_cuda:
            raise ValueError(f"{what} tensors must be CUDA tensors")
    raise ValueError(f"{what} tensors must be on one device")


def _check_sizes(what: str, *sizes: int) -> None:
    for size in sizes:
        if size > _MAX_SIZE:
            raise ValueError(f"{what} sizes must be at most {_MAX_SIZE}")


def _launch(symbol: str, on: torch.Tensor, *args) -> None:
    """One library call on the current stream of ``on``'s device."""
    library = bindings._LIBRARY or bindings._library()
    if on.get_device() == _current_device():
        code = library.functions[symbol](*args, _stream(on))
    else:
        with torch.cuda.device(on.device):
            code = library.functions[symbol](*args, _stream(on))
    if code:
        library.check(code)


# ---------------------------------------------------------------- quantisation


# The calls are host-bound at small sizes, so an operator's checks are first one
# expression that reads each attribute once; where it does not hold, the checks
# run one by one and raise.  The allocating forms do not check what they made.

_ROWS = {torch.bfloat16: "cuda_operator_quantize_fp8_block128_bf16",
         torch.float32: "cuda_operator_quantize_fp8_block128_f32"}
_TILES = {torch.bfloat16: "cuda_operator_quantize_fp8_block128_weight_bf16",
          torch.float32: "cuda_operator_quantize_fp8_block128_weight_f32"}


def _check_source(what: str, x: torch.Tensor) -> None:
    if x.dtype not in _ROWS:
        raise TypeError(f"{what} expects a bfloat16 or float32 input")


def _check_quantized(what: str, x: torch.Tensor, q: torch.Tensor, scale: torch.Tensor,
                     scale_shape: tuple[int, ...]) -> None:
    if q.shape != x.shape:
        raise ValueError(f"{what} output shape must be {tuple(x.shape)}")
    if scale.shape != scale_shape:
        raise ValueError(f"{what} scale shape must be {scale_shape}")
    if q.dtype != _E4M3 or scale.dtype != torch.float32:
        raise TypeError(f"{what} writes float8_e4m3fn values and float32 scales")


def _check_rows(x: torch.Tensor) -> tuple[int, int]:
    if x.ndim != 2:
        raise ValueError("x must be 2-D")
    _check_source("FP8 quantize", x)
    m, k = x.shape
    _check_sizes("FP8 quantize", m, k)
    return m, k


def quantize_fp8_block128_into(x: torch.Tensor, q: torch.Tensor,
                               scale: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows [M, K] (bf16 or fp32) to e4m3 [M, K] and fp32 scales [M, ceil(K/128)]."""
    m, k = _check_rows(x)
    _check_quantized("FP8 quantize", x, q, scale, (m, _blocks(k)))
    _check_placement("FP8 quantize", x, q, scale)
    if m and k:
        _launch(_ROWS[x.dtype], x, _ptr(x), _ptr(q), _ptr(scale), m, k)
    return q, scale


def quantize_fp8_block128(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Allocating form of :func:`quantize_fp8_block128_into`: ``(q, scale)``."""
    symbol = _ROWS.get(x.dtype)
    if symbol is None or x.ndim != 2 or not x.is_cuda or not x.is_contiguous():
        _check_rows(x)
        _check_placement("FP8 quantize", x)
    m, k = x.shape
    if m > _MAX_SIZE or k > _MAX_SIZE:
        _check_sizes("FP8 quantize", m, k)
    q = torch.empty_like(x, dtype=_E4M3)
    scale = torch.empty(m, _blocks(k), device=x.device, dtype=torch.float32)
    if m and k:
        _launch(symbol, x, x.data_ptr(), q.data_ptr(), scale.data_ptr(), m, k)
    return q, scale


def _weight_scale_shape(shape: torch.Size) -> tuple[int, ...]:
    return (*shape[:-2], _blocks(shape[-2]), _blocks(shape[-1]))


def _check_weight(weight: torch.Tensor) -> tuple[int, int, int]:
    if weight.ndim not in (2, 3):
        raise ValueError("weight must be 2-D or 3-D")
    _check_source("FP8 weight quantize", weight)
    n, k = weight.shape[-2:]
    experts = weight.shape[0] if weight.ndim == 3 else 1
    _check_sizes("FP8 weight quantize", n, k, experts * _blocks(n) * _blocks(k))
    return experts, n, k


def quantize_fp8_block128_weight_into(weight: torch.Tensor, q: torch.Tensor,
                                      scale: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Weights [N, K] or [E, N, K] (bf16 or fp32) to e4m3 and fp32 scales of 128 x 128 tiles.

    ``scale`` is [ceil(N/128), ceil(K/128)], with E in front where the weight has it.
    """
    what = "FP8 weight quantize"
    experts, n, k = _check_weight(weight)
    _check_quantized(what, weight, q, scale, _weight_scale_shape(weight.shape))
    _check_placement(what, weight, q, scale)
    if experts and n and k:
        _launch(_TILES[weight.dtype], weight, _ptr(weight), _ptr(q), _ptr(scale), experts, n, k)
    return q, scale


def quantize_fp8_block128_weight(weight: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Allocating form of :func:`quantize_fp8_block128_weight_into`: ``(q, scale)``."""
    experts, n, k = _check_weight(weight)
    _check_placement("FP8 weight quantize", weight)
    q = torch.empty_like(weight, dtype=_E4M3)
    scale = weight.new_empty(_weight_scale_shape(weight.shape), dtype=torch.float32)
    if experts and n and k:
        _launch(_TILES[weight.dtype], weight, _ptr(weight), _ptr(q), _ptr(scale), experts, n, k)
    return q, scale


# ---------------------------------------------------------------- products


def _check_fp8_operands(what: str, x_fp8: torch.Tensor, x_scale: torch.Tensor,
                        weight_fp8: torch.Tensor, weight_scale: torch.Tensor,
                        swiglu: bool) -> tuple[int, int, int]:
    """Shapes and types shared by the dense and the grouped products; returns (rows, k, n)."""
    m, k = x_fp8.shape
    w_shape = weight_fp8.shape
    w_rows = w_shape[-2]
    blocks = _blocks(k)
    if len(w_shape) == 2:
        scale_shape = (_blocks(w_rows), blocks)
    else:
        scale_shape = (w_shape[0], _blocks(w_rows), blocks)
    if (w_shape[-1] == k and k > 0 and not (swiglu and w_rows % (2 * BLOCK))
            and x_scale.shape == (m, blocks) and weight_scale.shape == scale_shape
            and x_fp8.dtype is _E4M3 and weight_fp8.dtype is _E4M3
            and x_scale.dtype is torch.float32 and weight_scale.dtype is torch.float32
            and m <= _MAX_SIZE and k <= _MAX_SIZE and w_rows <= _MAX_SIZE):
        return m, k, w_rows // 2 if swiglu else w_rows
    if w_shape[-1] != k:
        raise ValueError("x.shape[1] must equal the weight's last dimension")
    if k == 0:
        raise ValueError(f"{what} requires k > 0")
    if swiglu and w_rows % (2 * BLOCK):
        raise ValueError(f"{what} needs gate and up rows in whole blocks of {BLOCK}")
    if x_scale.shape != (m, blocks):
        raise ValueError(f"x scale shape must be {(m, blocks)}")
    if weight_scale.shape != scale_shape:
        raise ValueError(f"weight scale shape must be {scale_shape}")
    if x_fp8.dtype != _E4M3 or weight_fp8.dtype != _E4M3:
        raise TypeError(f"{what} expects float8_e4m3fn x and weight")
    if x_scale.dtype != torch.float32 or weight_scale.dtype != torch.float32:
        raise TypeError(f"{what} expects float32 scales")
    raise ValueError(f"{what} sizes must be at most {_MAX_SIZE}")


def _check_output(what: str, out: torch.Tensor, shape: tuple[int, ...]) -> None:
    if out.shape != shape:
        raise ValueError(f"output shape must be {shape}")
    if out.dtype != torch.bfloat16:
        raise TypeError(f"{what} expects a bfloat16 output")


def _gemm(swiglu: bool, x_fp8: torch.Tensor, x_scale: torch.Tensor, weight_fp8: torch.Tensor,
          weight_scale: torch.Tensor, out: torch.Tensor | None) -> torch.Tensor:
    what = "FP8 GEMM SwiGLU" if swiglu else "FP8 GEMM"
    if x_fp8.ndim != 2 or weight_fp8.ndim != 2:
        raise ValueError("x and weight must be 2-D")
    m, k, n = _check_fp8_operands(what, x_fp8, x_scale, weight_fp8, weight_scale, swiglu)
    if out is None:
        _check_placement(what, x_fp8, x_scale, weight_fp8, weight_scale)
        out = torch.empty(m, n, device=x_fp8.device, dtype=torch.bfloat16)
    else:
        _check_output(what, out, (m, n))
        _check_placement(what, x_fp8, x_scale, weight_fp8, weight_scale, out)
    if m and n:
        symbol = "cuda_operator_gemm_swiglu_fp8_block128" if swiglu else "cuda_operator_gemm_fp8_block128"
        _launch(symbol, x_fp8, _ptr(x_fp8), _ptr(x_scale), _ptr(weight_fp8), _ptr(weight_scale),
                _ptr(out), m, k, n)
    return out


def gemm_fp8_block128_into(x_fp8: torch.Tensor, x_scale: torch.Tensor, weight_fp8: torch.Tensor,
                           weight_scale: torch.Tensor, out_bf16: torch.Tensor) -> torch.Tensor:
    """bf16(x @ W.T) of block-scaled e4m3 x [M, K] and W [N, K], products and sums in fp32."""
    return _gemm(False, x_fp8, x_scale, weight_fp8, weight_scale, out_bf16)


def gemm_fp8_block128(x_fp8: torch.Tensor, x_scale: torch.Tensor, weight_fp8: torch.Tensor,
                      weight_scale: torch.Tensor) -> torch.Tensor:
    """Allocating form of :func:`gemm_fp8_block128_into`."""
    return _gemm(False, x_fp8, x_scale, weight_fp8, weight_scale, None)


def gemm_swiglu_fp8_block128_into(x_fp8: torch.Tensor, x_scale: torch.Tensor,
                                  packed_weight_fp8: torch.Tensor, weight_scale: torch.Tensor,
                                  out_bf16: torch.Tensor) -> torch.Tensor:
    """Packed form: bf16(silu(x @ Wg.T) * (x @ Wu.T)), packed_weight_fp8 [2N, K], gate rows first.

    N must be a multiple of 128, so that no tile of scales spans gate and up rows.
    """
    return _gemm(True, x_fp8, x_scale, packed_weight_fp8, weight_scale, out_bf16)


def gemm_swiglu_fp8_block128(x_fp8: torch.Tensor, x_scale: torch.Tensor,
                             packed_weight_fp8: torch.Tensor,
                             weight_scale: torch.Tensor) -> torch.Tensor:
    """Allocating form of :func:`gemm_swiglu_fp8_block128_into`."""
    return _gemm(True, x_fp8, x_scale, packed_weight_fp8, weight_scale, None)
