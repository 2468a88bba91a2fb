"""Matrix products grouped by expert, with ragged group sizes.

Rows of ``x`` [T, K] are sorted by expert: ``offsets``, an int32 CUDA tensor
[E + 1] that does not decrease, gives expert ``e`` the rows ``offsets[e]`` to
``offsets[e + 1]``.  It is read on the device alone, so a call never waits for
the GPU and can be captured in a CUDA graph and replayed with other offsets.
An expert may have no rows.  Rows of no expert (before ``offsets[0]``, from
``offsets[E]`` on, e.g. a batch padded to a fixed T) are neither used nor
written: the ``_into`` forms leave them as they were, the allocating forms
return them undefined.  Offsets outside [0, T] are clamped into it, so a wrong
array gives wrong rows but no access out of range.

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
from .fp8 import _check_fp8_operands, _check_placement, _check_sizes, _launch

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


def _check_ranks(x: torch.Tensor, weight: torch.Tensor) -> None:
    if x.ndim != 2 or weight.ndim != 3:
        raise ValueError("x must be 2-D and weight 3-D")


# ---------------------------------------------------------------- bf16


def _forward_into(swiglu: bool, x: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor,
                  out: torch.Tensor) -> torch.Tensor:
    what = "grouped GEMM SwiGLU" if swiglu else "grouped GEMM"
    _check_ranks(x, weight)
    t, k = x.shape
    experts, w_rows, _ = weight.shape
    if weight.shape[2] != k:
        raise ValueError("x.shape[1] must equal weight.shape[2]")
    if k == 0:
        raise ValueError(f"{what} requires k > 0")
    if swiglu and w_rows % 2:
        raise ValueError("packed weight must have an even number of rows")
    n = w_rows // 2 if swiglu else w_rows
    if out.shape != (t, n):
        raise ValueError(f"output shape must be {(t, n)}")
    _check_offsets(what, offsets, experts)
    _check_bf16(what, x, weight, out)
    _check_sizes(what, t, k, w_rows)
    _check_placement(what, x, weight, offsets, out)
    if t and n and experts:
        symbol = "cuda_operator_gemm_grouped_swiglu_bf16" if swiglu else "cuda_operator_gemm_grouped_bf16"
        _launch(symbol, x, _ptr(x), _ptr(weight), _ptr(offsets), _ptr(out), t, k, n, experts)
    return out


def gemm_grouped_bf16_into(x_bf16: torch.Tensor, weight_bf16: torch.Tensor, offsets: torch.Tensor,
                           out_bf16: torch.Tensor) -> torch.Tensor:
    """bf16(x[r] @ W[e].T) for the rows r of each expert e; x [T, K], W [E, N, K], out [T, N]."""
    return _forward_into(False, x_bf16, weight_bf16, offsets, out_bf16)


def gemm_grouped_bf16(x_bf16: torch.Tensor, weight_bf16: torch.Tensor,
                      offsets: torch.Tensor) -> torch.Tensor:
    """Allocating form of :func:`gemm_grouped_bf16_into`."""
    _check_ranks(x_bf16, weight_bf16)
    out = torch.empty((x_bf16.shape[0], weight_bf16.shape[1]), device=x_bf16.device,
                      dtype=torch.bfloat16)
    return gemm_grouped_bf16_into(x_bf16, weight_bf16, offsets, out)


def gemm_grouped_swiglu_bf16_into(x_bf16: torch.Tensor, packed_weight_bf16: torch.Tensor,
                                  offsets: torch.Tensor, out_bf16: torch.Tensor) -> torch.Tensor:
    """bf16(silu(x[r] @ Wg[e].T) * (x[r] @ Wu[e].T)); packed weight [E, 2N, K], gate rows first."""
    return _forward_into(True, x_bf16, packed_weight_bf16, offsets, out_bf16)


def gemm_grouped_swiglu_bf16(x_bf16: torch.Tensor, packed_weight_bf16: torch.Tensor,
                             offsets: torch.Tensor) -> torch.Tensor:
    """Allocating form of :func:`gemm_grouped_swiglu_bf16_into`."""
    _check_ranks(x_bf16, packed_weight_bf16)
    out = torch.empty((x_bf16.shape[0], packed_weight_bf16.shape[1] // 2), device=x_bf16.device,
                      dtype=torch.bfloat16)
    return gemm_grouped_swiglu_bf16_into(x_bf16, packed_weight_bf16, offsets, out)


# ---------------------------------------------------------------- bf16 gradients


def _check_grad_input(grad: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor,
                      out: torch.Tensor) -> None:
    what = "grouped GEMM gradient"
    _check_ranks(grad, weight)
    t, n = grad.shape
    experts, _, k = weight.shape
    if weight.shape[1] != n:
        raise ValueError("grad.shape[1] must equal weight.shape[1]")
    if n == 0:
        raise ValueError(f"{what} requires n > 0")
    if out.shape != (t, k):
        raise ValueError(f"output shape must be {(t, k)}")
    _check_offsets(what, offsets, experts)
    _check_bf16(what, grad, weight, out)
    _check_sizes(what, t, k, n)


def _run_grad_input(grad: torch.Tensor, weight: torch.Tensor, offsets: torch.Tensor,
                    out: torch.Tensor) -> torch.Tensor:
    t, n = grad.shape
    experts, _, k = weight.shape
    if t and k and experts:
        _launch("cuda_operator_gemm_grouped_bf16_grad_input", grad, _ptr(grad), _ptr(weight),
                _ptr(offsets), _ptr(out), t, k, n, experts)
    return out


def gemm_grouped_bf16_grad_input_into(grad_bf16: torch.Tensor, weight_bf16: torch.Tensor,
                                      offsets: torch.Tensor,
                                      grad_input_bf16: torch.Tensor) -> torch.Tensor:
    """Gradient of :func:`gemm_grouped_bf16` by x: bf16(grad[r] @ W[e]); grad [T, N], out [T, K]."""
    _check_grad_input(grad_bf16, weight_bf16, offsets, grad_input_bf16)
    _check_placement("grouped GEMM gradient", grad_bf16, weight_bf16, offsets, grad_input_bf16)
    return _run_grad_input(grad_bf16, weight_bf16, offsets, grad_input_bf16)


def gemm_grouped_bf16_grad_input(grad_bf16: torch.Tensor, weight_bf16: torch.Tensor,
                                 offsets: torch.Tensor) -> torch.Tensor:
    """Allocating form of :func:`gemm_grouped_bf16_grad_input_into`."""
    _check_ranks(grad_bf16, weight_bf16)
    out = torch.empty((grad_bf16.shape[0], weight_bf16.shape[2]), device=grad_bf16.device,
                      dtype=torch.bfloat16)
    return gemm_grouped_bf16_grad_input_into(grad_bf16, weight_bf16, offsets, out)


def _check_grad_weight(grad: torch.Tensor, x: torch.Tensor, offsets: torch.Tensor,
                       out: torch.Tensor) -> None:
    what = "grouped GEMM gradient"
    if grad.ndim != 2 or x.ndim != 2 or out.ndim != 3:
        raise ValueError("grad and x must be 2-D and the output 3-D")
    t, n = grad.shape
    k = x.shape[1]
    if x.shape[0] != t:
        raise ValueError("grad and x must have the same number of rows")
    experts = out.shape[0]
    if out.shape != (experts, n, k):
        raise ValueError(f"output shape must be {(experts, n, k)}")
    _check_offsets(what, offsets, experts)
    _check_bf16(what, grad, x, out)
    _check_sizes(what, t, k, n)


def _run_grad_weight(grad: torch.Tensor, x: torch.Tensor, offsets: torch.Tensor,
                     out: torch.Tensor) -> torch.Tensor:
    experts, n, k = out.shape
    if n and k and experts:
        _launch("cuda_operator_gemm_grouped_bf16_grad_weight", grad, _ptr(grad), _ptr(x),
                _ptr(offsets), _ptr(out), grad.shape[0], k, n, experts)
    return out


def gemm_grouped_bf16_grad_weight_into(grad_bf16: torch.Tensor, x_bf16: torch.Tensor,
                                       offsets: torch.Tensor,
                                       grad_weight_bf16: torch.Tensor) -> torch.Tensor:
    """Gradient of :func:`gemm_grouped_bf16` by W: bf16(grad[rows of e].T @ x[rows of e]).

    grad [T, N], x [T, K], out [E, N, K], which is written whole: zeros for an
    expert without rows.
    """
    _check_grad_weight(grad_bf16, x_bf16, offsets, grad_weight_bf16)
    _check_placement("grouped GEMM gradient", grad_bf16, x_bf16, offsets, grad_weight_bf16)
    return _run_grad_weight(grad_bf16, x_bf16, offsets, grad_weight_bf16)


def gemm_grouped_bf16_grad_weight(grad_bf16: torch.Tensor, x_bf16: torch.Tensor,
                                  offsets: torch.Tensor) -> torch.Tensor:
    """Allocating form of :func:`gemm_grouped_bf16_grad_weight_into`."""
    if grad_bf16.ndim != 2 or x_bf16.ndim != 2:
        raise ValueError("grad and x must be 2-D and the output 3-D")
    if offsets.ndim != 1 or offsets.shape[0] == 0:
        raise ValueError("offsets must be 1-D with one entry more than there are experts")
    out = torch.empty((offsets.shape[0] - 1, grad_bf16.shape[1], x_bf16.shape[1]),
                      device=grad_bf16.device, dtype=torch.bfloat16)
    return gemm_grouped_bf16_grad_weight_into(grad_bf16, x_bf16, offsets, out)


def gemm_grouped_bf16_backward(grad_bf16: torch.Tensor, x_bf16: torch.Tensor,
                               weight_bf16: torch.Tensor,
                               offsets: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Both gradients of :func:`gemm_grouped_bf16`: ``(grad_input, grad_weight)``."""
    _check_ranks(x_bf16, weight_bf16)
    grad_input = torch.empty(x_bf16.shape, device=x_bf16.device, dtype=torch.bfloat16)
    grad_weight = torch.empty(weight_bf16.shape, device=x_bf16.device, dtype=torch.bfloat16)
    _check_grad_weight(grad_bf16, x_bf16, offsets, grad_weight)
    _check_grad_input(grad_bf16, weight_bf16, offsets, grad_input)
    _check_placement("grouped GEMM gradient", grad_bf16, x_bf16, weight_bf16, offsets)
    return (_run_grad_input(grad_bf16, weight_bf16, offsets, grad_input),
            _run_grad_weight(grad_bf16, x_bf16, offsets, grad_weight))


# ---------------------------------------------------------------- block-scaled e4m3


def _fp8_into(swiglu: bool, x_fp8: torch.Tensor, x_scale: torch.Tensor, weight_fp8: torch.Tensor,
              weight_scale: torch.Tensor, offsets: torch.Tensor,
              out: torch.Tensor) -> torch.Tensor:
    what = "grouped FP8 GEMM SwiGLU" if swiglu else "grouped FP8 GEMM"
    _check_ranks(x_fp8, weight_fp8)
    experts = weight_fp8.shape[0]
    t, k, n = _check_fp8_operands(what, x_fp8, x_scale, weight_fp8, weight_scale, out, swiglu)
    _check_offsets(what, offsets, experts)
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
    return _fp8_into(False, x_fp8, x_scale, weight_fp8, weight_scale, offsets, out_bf16)


def gemm_grouped_fp8_block128(x_fp8: torch.Tensor, x_scale: torch.Tensor,
                              weight_fp8: torch.Tensor, weight_scale: torch.Tensor,
                              offsets: torch.Tensor) -> torch.Tensor:
    """Allocating form of :func:`gemm_grouped_fp8_block128_into`."""
    _check_ranks(x_fp8, weight_fp8)
    out = torch.empty((x_fp8.shape[0], weight_fp8.shape[1]), device=x_fp8.device,
                      dtype=torch.bfloat16)
    return gemm_grouped_fp8_block128_into(x_fp8, x_scale, weight_fp8, weight_scale, offsets, out)


def gemm_grouped_swiglu_fp8_block128_into(x_fp8: torch.Tensor, x_scale: torch.Tensor,
                                          packed_weight_fp8: torch.Tensor,
                                          weight_scale: torch.Tensor, offsets: torch.Tensor,
                                          out_bf16: torch.Tensor) -> torch.Tensor:
    """:func:`gemm_grouped_swiglu_bf16_into` of block-scaled e4m3 operands; N % 128 == 0."""
    return _fp8_into(True, x_fp8, x_scale, packed_weight_fp8, weight_scale, offsets, out_bf16)


def gemm_grouped_swiglu_fp8_block128(x_fp8: torch.Tensor, x_scale: torch.Tensor,
                                     packed_weight_fp8: torch.Tensor, weight_scale: torch.Tensor,
                                     offsets: torch.Tensor) -> torch.Tensor:
    """Allocating form of :func:`gemm_grouped_swiglu_fp8_block128_into`."""
    _check_ranks(x_fp8, packed_weight_fp8)
    out = torch.empty((x_fp8.shape[0], packed_weight_fp8.shape[1] // 2), device=x_fp8.device,
                      dtype=torch.bfloat16)
    return gemm_grouped_swiglu_fp8_block128_into(x_fp8, x_scale, packed_weight_fp8, weight_scale,
                                                 offsets, out)
