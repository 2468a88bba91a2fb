"""Matrix products grouped by expert, with ragged group sizes.

Rows of ``x`` [T, K] are sorted by expert: ``offsets``, an int32 CUDA tensor
[E + 1] that does not decrease, gives expert ``e`` the rows ``offsets[e]`` to
``offsets[e + 1]``.  It is read on the device alone, so a call never waits for
the GPU and can be captured in a CUDA graph and replayed with other offsets.
An expert may have no rows.  Rows of no expert (before ``offsets[0]``, from
``offsets[E]`` on, e.g. a batch padded to a fixed T) are neither used nor
written: the ``_into`` forms leave them as they were, the allocating forms
return them undefined.  An offset outside [0, T] is clamped into it and one
below an earlier offset counts as that one, so a wrong array gives wrong rows
but no access out of range.

Weights are [E, N, K]; the SwiGLU forms take [E, 2N, K] with the N gate rows
first, as the dense packed GEMM+SwiGLU does.  Sums are fp32 and outputs bf16.
The bf16 form has both gradients; nothing here records for autograd.  The
products run on the tensor cores where rows are whole multiples of 16 bytes
(K, and for the gradients N, a multiple of 8; for e4m3 K a multiple of 16) and
the operands start on 16-byte boundaries, elsewhere on a much slower
CUDA-core kernel.
"""

from __future__ import annotations

import torch

from .bindings import _ptr
from .fp8 import (_MAX_SIZE, _check_fp8_operands, _check_output, _check_placement, _check_sizes,
                  _launch)

__all__ = [
    "gemm_grouped_bf16", "gemm_grouped_bf16_into",
    "gemm_grouped_swiglu_bf16", "gemm_grouped_swiglu_bf16_into",
    "gemm_grouped_bf16_grad_input", "gemm_grouped_bf16_grad_input_into",
    "gemm_grouped_bf16_grad_weight", "gemm_grouped_bf16_grad_weight_into",
    "gemm_grouped_bf16_backward",
    "gemm_grouped_fp8_block128", "gemm_grouped_fp8_block128_into",
    "gemm_grouped_swiglu_fp8_block128", "gemm_grouped_swiglu_fp8_block128_into",
]

#: Most experts of one call.
MAX_EXPERTS = 1024


def _check_offsets(what: str, offsets: torch.Tensor, experts: int) -> None:
    if experts > MAX_EXPERTS:
        raise ValueError(f"{what} takes at most {MAX_EXPERTS} experts")
    if offsets.ndim != 1 or offsets.shape[0] != experts + 1:
        raise ValueError(f"offsets must have shape ({experts + 1},)")
    if offsets.dtype != torch.int32:
        raise TypeError(f"{what} expects int32 offsets")


def _check_bf16(what: str, *tensors: torch.Tensor) -> None:
    for t in tensors:
        if t.dtype != torch.bfloat16:
            raise TypeError(f"{what} expects bfloat16 tensors")


def _new(on: torch.Tensor, *shape: int) -> torch.Tensor:
    return torch.empty(*shape, device=on.device, dtype=torch.bfloat16)


def _check_ranks(x: torch.Tensor, weight: torch.Tensor) -> None:
    if x.ndim != 2 or weight.ndim != 3:
        raise ValueError("x must be 2-D and weight 3-D")


# ---------------------------------------------------------------- bf16


def _check_forward(what: str, swiglu: bool, x: torch.Tensor, weight: torch.Tensor,
                   offsets: torch.Tensor) -> tuple[int, int, int, int]:
    """Checks of all but the output and the placement; returns (t, k, n, experts)."""
    _check_ranks(x, weight)
    t, k = x.shape
    experts, w_rows, w_cols = weight.shape
    n = w_rows // 2 if swiglu else w_rows
    if (w_cols == k and k > 0 and not (swiglu and w_rows % 2)
            and offsets.shape == (experts + 1,) and offsets.dtype is torch.int32
            and x.dtype is torch.bfloat16 and weight.dtype is torch.bfloat16
            and experts <= MAX_EXPERTS and t <= _MAX_SIZE and k <= _MAX_SIZE
            and w_rows <= _MAX_SIZE):
        return t, k, n, experts
    if w_cols != k:
        raise ValueError("x.shape[1] must equal weight.shape[2]")
    if k == 0:
        raise ValueError(f"{what} requires k > 0")
    if swiglu and w_rows % 2:
        raise ValueError("packed weight must have an even number of rows")
    _check_offsets(what, offsets, experts)
    _check_bf16(what, x, weight)
    _check_sizes(what, t, k, w_rows)
    raise AssertionError("unreachable")


def _forward(swiglu: bool, x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor,
             out: torch.Tensor | None) -> torch.Tensor:
    what = "grouped GEMM SwiGLU" if swiglu else "grouped GEMM"
    t, k, n, experts = _check_forward(what, swiglu, x, weight, offsets)
    if out is None:
        _check_placement(what, x, weight, offsets)
        out = _new(x, t, n)
    else:
        _check_output(what, out, (t, n))
        _check_placement(what, x, weight, offsets, out)
    if t and n and experts:
        symbol = "cuda_operator_gemm_grouped_swiglu_bf16" if swiglu else "cuda_operator_gemm_grouped_bf16"
        _launch(symbol, x, _ptr(x), _ptr(weight), _ptr(offsets), _ptr(out), t, k, n, experts)
    return out


def gemm_grouped_bf16_into(x_bf16: torch.Tensor, weight_bf16: torch.Tensor, offsets: torch.Tensor,
                           out_bf16: torch.Tensor) -> torch.Tensor:
    """bf16(x[r] @ W[e].T) for the rows r of each expert e; x [T, K], W [E, N, K], out [T, N]."""
    return _forward(False, x_bf16, weight_bf16, offsets, out_bf16)


def gemm_grouped_bf16(x_bf16: torch.Tensor, weight_bf16: torch.Tensor,
                      offsets: torch.Tensor) -> torch.Tensor:
    """Allocating form of :func:`gemm_grouped_bf16_into`."""
    return _forward(False, x_bf16, weight_bf16, offsets, None)


def gemm_grouped_swiglu_bf16_into(x_bf16: torch.Tensor, packed_weight_bf16: torch.Tensor,
                                  offsets: torch.Tensor, out_bf16: torch.Tensor) -> torch.Tensor:
    """bf16(silu(x[r] @ Wg[e].T) * (x[r] @ Wu[e].T)); packed weight [E, 2N, K], gate rows first."""
    return _forward(True, x_bf16, packed_weight_bf16, offsets, out_bf16)


def gemm_grouped_swiglu_bf16(x_bf16: torch.Tensor, packed_weight_bf16: torch.Tensor,
                             offsets: torch.Tensor) -> torch.Tensor:
    """Allocating form of :func:`gemm_grouped_swiglu_bf16_into`."""
    return _forward(True, x_bf16, packed_weight_bf16, offsets, None)


# ---------------------------------------------------------------- bf16 gradients


_GRAD = "grouped GEMM gradient"


def _check_grad_input(grad: torch.Tensor, weight: torch.Tensor,
                      offsets: torch.Tensor) -> tuple[int, int, int, int]:
    _check_ranks(grad, weight)
    t, n = grad.shape
    experts, w_rows, k = weight.shape
    if w_rows != n:
        raise ValueError("grad.shape[1] must equal weight.shape[1]")
    if n == 0:
        raise ValueError(f"{_GRAD} requires n > 0")
    _check_offsets(_GRAD, offsets, experts)
    _check_bf16(_GRAD, grad, weight)
    _check_sizes(_GRAD, t, k, n)
    return t, k, n, experts


def _run_grad_input(grad: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor,
                    out: torch.Tensor, t: int, k: int, n: int, experts: int) -> torch.Tensor:
    if t and k and experts:
        _launch("cuda_operator_gemm_grouped_bf16_grad_input", grad, _ptr(grad), _ptr(weight),
                _ptr(offsets), _ptr(out), t, k, n, experts)
    return out


def gemm_grouped_bf16_grad_input_into(grad_bf16: torch.Tensor, weight_bf16: torch.Tensor,
                                      offsets: torch.Tensor,
                                      grad_input_bf16: torch.Tensor) -> torch.Tensor:
    """Gradient of :func:`gemm_grouped_bf16` by x: bf16(grad[r] @ W[e]); grad [T, N], out [T, K]."""
    t, k, n, experts = _check_grad_input(grad_bf16, weight_bf16, offsets)
    _check_output(_GRAD, grad_input_bf16, (t, k))
    _check_placement(_GRAD, grad_bf16, weight_bf16, offsets, grad_input_bf16)
    return _run_grad_input(grad_bf16, weight_bf16, offsets, grad_input_bf16, t, k, n, experts)


def gemm_grouped_bf16_grad_input(grad_bf16: torch.Tensor, weight_bf16: torch.Tensor,
                                 offsets: torch.Tensor) -> torch.Tensor:
    """Allocating form of :func:`gemm_grouped_bf16_grad_input_into`."""
    t, k, n, experts = _check_grad_input(grad_bf16, weight_bf16, offsets)
    _check_placement(_GRAD, grad_bf16, weight_bf16, offsets)
    return _run_grad_input(grad_bf16, weight_bf16, offsets, _new(grad_bf16, t, k), t, k, n, experts)


def _check_grad_weight(grad: torch.Tensor, x: torch.Tensor,
                       offsets: torch.Tensor) -> tuple[int, int, int, int]:
    if grad.ndim != 2 or x.ndim != 2:
        raise ValueError("grad and x must be 2-D")
    if offsets.ndim != 1 or offsets.shape[0] == 0:
        raise ValueError("offsets must be 1-D with one entry more than there are experts")
    t, n = grad.shape
    rows, k = x.shape
    if rows != t:
        raise ValueError("grad and x must have the same number of rows")
    experts = offsets.shape[0] - 1
    _check_offsets(_GRAD, offsets, experts)
    _check_bf16(_GRAD, grad, x)
    _check_sizes(_GRAD, t, k, n)
    return t, k, n, experts


def _run_grad_weight(grad: torch.Tensor, x: torch.Tensor, offsets: torch.Tensor,
                     out: torch.Tensor, t: int, k: int, n: int, experts: int) -> torch.Tensor:
    if n and k and experts:
        _launch("cuda_operator_gemm_grouped_bf16_grad_weight", grad, _ptr(grad), _ptr(x),
                _ptr(offsets), _ptr(out), t, k, n, experts)
    return out


def gemm_grouped_bf16_grad_weight_into(grad_bf16: torch.Tensor, x_bf16: torch.Tensor,
                                       offsets: torch.Tensor,
                                       grad_weight_bf16: torch.Tensor) -> torch.Tensor:
    """Gradient of :func:`gemm_grouped_bf16` by W: bf16(grad[rows of e].T @ x[rows of e]).

    grad [T, N], x [T, K], out [E, N, K], which is written whole: zeros for an
    expert without rows.
    """
    t, k, n, experts = _check_grad_weight(grad_bf16, x_bf16, offsets)
    _check_output(_GRAD, grad_weight_bf16, (experts, n, k))
    _check_placement(_GRAD, grad_bf16, x_bf16, offsets, grad_weight_bf16)
    return _run_grad_weight(grad_bf16, x_bf16, offsets, grad_weight_bf16, t, k, n, experts)


def gemm_grouped_bf16_grad_weight(grad_bf16: torch.Tensor, x_bf16: torch.Tensor,
                                  offsets: torch.Tensor) -> torch.Tensor:
    """Allocating form of :func:`gemm_grouped_bf16_grad_weight_into`."""
    t, k, n, experts = _check_grad_weight(grad_bf16, x_bf16, offsets)
    _check_placement(_GRAD, grad_bf16, x_bf16, offsets)
    return _run_grad_weight(grad_bf16, x_bf16, offsets, _new(grad_bf16, experts, n, k), t, k,
                            n, experts)


def gemm_grouped_bf16_backward(grad_bf16: torch.Tensor, x_bf16: torch.Tensor,
                               weight_bf16: torch.Tensor,
                               offsets: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Both gradients of :func:`gemm_grouped_bf16`: ``(grad_input, grad_weight)``."""
    t, k, n, experts = _check_grad_input(grad_bf16, weight_bf16, offsets)
    if x_bf16.shape != (t, k):
        raise ValueError(f"x shape must be {(t, k)}")
    _check_bf16(_GRAD, x_bf16)
    _check_placement(_GRAD, grad_bf16, x_bf16, weight_bf16, offsets)
    grad_input = _new(grad_bf16, t, k)
    grad_weight = _new(grad_bf16, experts, n, k)
    if k and experts:
        _launch("cuda_operator_gemm_grouped_bf16_backward", grad_bf16, _ptr(grad_bf16),
                _ptr(x_bf16), _ptr(weight_bf16), _ptr(offsets), _ptr(grad_input),
                _ptr(grad_weight), t, k, n, experts)
    return grad_input, grad_weight


# ---------------------------------------------------------------- block-scaled e4m3


def _fp8(swiglu: bool, x_fp8: torch.Tensor, x_scale: torch.Tensor, weight_fp8: torch.Tensor,
         weight_scale: torch.Tensor, offsets: torch.Tensor,
         out: torch.Tensor | None) -> torch.Tensor:
    what = "grouped FP8 GEMM SwiGLU" if swiglu else "grouped FP8 GEMM"
    _check_ranks(x_fp8, weight_fp8)
    experts = weight_fp8.shape[0]
    t, k, n = _check_fp8_operands(what, x_fp8, x_scale, weight_fp8, weight_scale, swiglu)
    _check_offsets(what, offsets, experts)
    if out is None:
        _check_placement(what, x_fp8, x_scale, weight_fp8, weight_scale, offsets)
        out = _new(x_fp8, t, n)
    else:
        _check_output(what, out, (t, n))
        _check_placement(what, x_fp8, x_scale, weight_fp8, weight_scale, offsets, out)
    if t and n and experts:
        symbol = ("cuda_operator_gemm_grouped_swiglu_fp8_block128" if swiglu
                  else "cuda_operator_gemm_grouped_fp8_block128")
        _launch(symbol, x_fp8, _ptr(x_fp8), _ptr(x_scale), _ptr(weight_fp8), _ptr(weight_scale),
                _ptr(offsets), _ptr(out), t, k, n, experts)
    return out


def gemm_grouped_fp8_block128_into(x_fp8: torch.Tensor, x_scale: torch.Tensor,
                                   weight_fp8: torch.Tensor, weight_scale: torch.Tensor,
                                   offsets: torch.Tensor, out_bf16: torch.Tensor) -> torch.Tensor:
    """:func:`gemm_grouped_bf16_into` of block-scaled e4m3 operands (see ``fp8``)."""
    return _fp8(False, x_fp8, x_scale, weight_fp8, weight_scale, offsets, out_bf16)


def gemm_grouped_fp8_block128(x_fp8: torch.Tensor, x_scale: torch.Tensor,
                              weight_fp8: torch.Tensor, weight_scale: torch.Tensor,
                              offsets: torch.Tensor) -> torch.Tensor:
    """Allocating form of :func:`gemm_grouped_fp8_block128_into`."""
    return _fp8(False, x_fp8, x_scale, weight_fp8, weight_scale, offsets, None)


def gemm_grouped_swiglu_fp8_block128_into(x_fp8: torch.Tensor, x_scale: torch.Tensor,
                                          packed_weight_fp8: torch.Tensor,
                                          weight_scale: torch.Tensor, offsets: torch.Tensor,
                                          out_bf16: torch.Tensor) -> torch.Tensor:
    """:func:`gemm_grouped_swiglu_bf16_into` of block-scaled e4m3 operands; N % 128 == 0."""
    return _fp8(True, x_fp8, x_scale, packed_weight_fp8, weight_scale, offsets, out_bf16)


def gemm_grouped_swiglu_fp8_block128(x_fp8: torch.Tensor, x_scale: torch.Tensor,
                                     packed_weight_fp8: torch.Tensor, weight_scale: torch.Tensor,
                                     offsets: torch.Tensor) -> torch.Tensor:
    """Allocating form of :func:`gemm_grouped_swiglu_fp8_block128_into`."""
    return _fp8(True, x_fp8, x_scale, packed_weight_fp8, weight_scale, offsets, None)
