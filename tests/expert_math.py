"""64-bit forms of the expert-layer operators and the error bounds of their results.

Bounds, for a sum of ``depth`` products with absolute sum ``s`` (sum of |a||b|):
a tensor core or an FMA chain keeps at least 24 bits of each partial sum, each
partial sum is at most ``s``, and an addition may truncate, so it is off by at
most ``2**-23 * s``: in all ``depth * 2**-23 * s``.  Block scales add a few
roundings of 2**-24 each (``depth + 8`` covers them).  The bf16 output is
rounded once more, by at most ``2**-8`` of its value (half a step).
"""

from __future__ import annotations

import torch

BLOCK = 128
AMAX_FLOOR = 2.0 ** -100
HALF_STEP_BF16 = torch.finfo(torch.bfloat16).eps / 2


def grid_e4m3(v: torch.Tensor) -> torch.Tensor:
    """64-bit values in [-448, 448] to the nearest e4m3 value, ties to even."""
    _, e = torch.frexp(v)
    step = torch.pow(2.0, (e.clamp(min=-5) - 4).double())
    return torch.round(v / step) * step


def spread(scale: torch.Tensor, height: int, n: int, k: int) -> torch.Tensor:
    """Scales of height x 128 blocks, one for each value of [..., n, k]."""
    rows = torch.arange(n, device=scale.device) // height
    cols = torch.arange(k, device=scale.device) // BLOCK
    return scale.double()[..., rows, :][..., cols]


def block_amax(v: torch.Tensor, height: int) -> torch.Tensor:
    """Largest magnitude (at least 2**-100) of each height x 128 block of [n, k]."""
    n, k = v.shape
    nb, kb = -(-n // height), -(-k // BLOCK)
    padded = torch.zeros((nb * height, kb * BLOCK), dtype=torch.float64, device=v.device)
    padded[:n, :k] = v.double().abs()
    return padded.view(nb, height, kb, BLOCK).amax((1, 3)).clamp(min=AMAX_FLOOR)


def quantize(v: torch.Tensor, height: int) -> tuple[torch.Tensor, torch.Tensor]:
    """(values before rounding to e4m3, scales) in 64 bits."""
    amax = block_amax(v, height)
    return v.double() * 448.0 / spread(amax, height, *v.shape), amax / 448.0


def product(x: torch.Tensor, w: torch.Tensor, swiglu: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """x @ w.T (or silu(gate) * up) of 64-bit operands, and the error bound of its bf16 result."""
    h = x @ w.mT
    err = (x.shape[1] + 8) * 2.0 ** -23 * (x.abs() @ w.abs().mT)
    if swiglu:
        n = h.shape[1] // 2
        g, u, eg, eu = h[:, :n], h[:, n:], err[:, :n], err[:, n:]
        silu = g * torch.sigmoid(g)
        h = silu * u
        # |d silu / d g| < 1.1; the activation's fp32 arithmetic (an exponential
        # and a division of a few units in the last place) is within 2**-19
        err = 1.1 * eg * (u.abs() + eu) + silu.abs() * eu + 2.0 ** -19 * h.abs()
    return h, err + HALF_STEP_BF16 * (h.abs() + err)


def assert_within(got: torch.Tensor, want: torch.Tensor, bound: torch.Tensor) -> None:
    got = got.double()
    assert got.shape == want.shape
    assert torch.isfinite(got).all()
    # 1e-38: a zero bound (an exact zero) still admits bf16's own underflow
    excess = (got - want).abs() - bound - 1e-38
    worst = float(excess.max()) if excess.numel() else 0.0
    assert worst <= 0.0, f"off by {worst} more than the bound at {int(excess.argmax())}"


def offsets_of(lengths: list[int], first: int = 0) -> torch.Tensor:
    out = [first]
    for n in lengths:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32)


def small_integers(shape, g: torch.Generator, most: int = 2) -> torch.Tensor:
    """Integers in [-most, most] as fp32: sums of few of them are exact in every type."""
    return torch.randint(-most, most + 1, shape, generator=g).float()
