"""One size at least for each tile shape that the expert-layer products run in on a B200 (148 SMs)."""

from __future__ import annotations

SM_COUNT = 148

PAIRS = (2, 256, 128, 1)
WIDE = (1, 256, 128, 1)
SINGLE = (1, 128, 128, 1)
FEW = (1, 128, 32, 1)
SHARED = {(columns, ctas): (1, columns, 32, ctas) for columns in (64, 128) for ctas in (2, 4)}

_BF16 = {PAIRS, WIDE, SINGLE, FEW, SHARED[128, 2], SHARED[128, 4]}
_FP8 = {PAIRS, WIDE, SINGLE, *SHARED.values()}

#: Every kernel that the library is compiled with, by product (None: two launches).
KERNELS = {
    "bf16": _BF16, "swiglu_bf16": _BF16, "grad_input": _BF16,
    "grad_weight": {PAIRS, WIDE, SINGLE},
    "both_grads": {FEW, SINGLE, None},
    "fp8": _FP8, "swiglu_fp8": _FP8, "dense_fp8": _FP8, "dense_swiglu_fp8": _FP8,
}

#: (product, tiles, rows, experts, n, k): odd rows, widths that end inside a tile,
#: sums that end inside a block of 64 (bf16) or 128 (e4m3).
CASES = [
    ("bf16", PAIRS, 5003, 5, 2000, 1032), ("bf16", WIDE, 1205, 11, 1528, 840),
    ("bf16", SINGLE, 701, 4, 776, 456), ("bf16", FEW, 67, 9, 1511, 1000),
    ("bf16", SHARED[128, 2], 35, 3, 1000, 712), ("bf16", SHARED[128, 4], 9, 3, 424, 2056),
    ("swiglu_bf16", PAIRS, 4001, 4, 1000, 1032), ("swiglu_bf16", WIDE, 1205, 11, 776, 840),
    ("swiglu_bf16", SINGLE, 701, 4, 388, 456), ("swiglu_bf16", FEW, 67, 9, 755, 1000),
    ("swiglu_bf16", SHARED[128, 2], 35, 3, 500, 712), ("swiglu_bf16", SHARED[128, 4], 9, 3, 212, 2056),
    ("grad_input", PAIRS, 5003, 5, 1032, 2000), ("grad_input", WIDE, 1205, 11, 840, 1528),
    ("grad_input", SINGLE, 701, 4, 456, 776), ("grad_input", FEW, 67, 9, 1000, 1512),
    ("grad_input", SHARED[128, 2], 35, 3, 712, 1000), ("grad_input", SHARED[128, 4], 9, 3, 2056, 424),
    ("grad_weight", PAIRS, 8071, 8, 2040, 2008), ("grad_weight", WIDE, 2053, 13, 1000, 1032),
    ("grad_weight", SINGLE, 211, 6, 136, 200),
    ("both_grads", FEW, 67, 9, 216, 184), ("both_grads", SINGLE, 1103, 20, 776, 520),
    ("both_grads", None, 8071, 8, 1032, 2008),
    ("fp8", PAIRS, 5003, 5, 2000, 1040), ("fp8", WIDE, 260, 37, 1016, 528),
    ("fp8", SINGLE, 701, 4, 776, 464), ("fp8", SHARED[64, 2], 35, 3, 424, 528),
    ("fp8", SHARED[64, 4], 9, 3, 212, 2064), ("fp8", SHARED[128, 2], 70, 3, 1500, 528),
    ("fp8", SHARED[128, 4], 9, 3, 1001, 2064),
    ("swiglu_fp8", PAIRS, 5003, 5, 1024, 1040), ("swiglu_fp8", WIDE, 260, 37, 512, 528),
    ("swiglu_fp8", SINGLE, 701, 4, 384, 464), ("swiglu_fp8", SHARED[64, 2], 35, 3, 256, 528),
    ("swiglu_fp8", SHARED[64, 4], 9, 3, 128, 2064), ("swiglu_fp8", SHARED[128, 2], 70, 3, 768, 528),
    ("swiglu_fp8", SHARED[128, 4], 9, 3, 512, 2064),
    ("dense_fp8", PAIRS, 4003, 1, 2000, 1040), ("dense_fp8", WIDE, 1028, 1, 3605, 208),
    ("dense_fp8", SINGLE, 301, 1, 1000, 2064), ("dense_fp8", SHARED[64, 2], 35, 1, 1500, 528),
    ("dense_fp8", SHARED[64, 4], 9, 1, 1000, 2064), ("dense_fp8", SHARED[128, 2], 70, 1, 2500, 528),
    ("dense_fp8", SHARED[128, 4], 9, 1, 4001, 2064),
    ("dense_swiglu_fp8", PAIRS, 4003, 1, 1024, 1040), ("dense_swiglu_fp8", WIDE, 529, 1, 3200, 208),
    ("dense_swiglu_fp8", SINGLE, 301, 1, 512, 2064), ("dense_swiglu_fp8", SHARED[64, 2], 35, 1, 640, 528),
    ("dense_swiglu_fp8", SHARED[64, 4], 9, 1, 512, 2064),
    ("dense_swiglu_fp8", SHARED[128, 2], 70, 1, 1280, 528),
    ("dense_swiglu_fp8", SHARED[128, 4], 9, 1, 2048, 2064),
]


def ragged(t: int, experts: int) -> list[int]:
    """Rows of each expert: uneven, every fifth without any, `t` in all."""
    share = [e % 5 for e in range(experts)] if experts > 1 else [1]
    lengths = [t * s // sum(share) for s in share]
    lengths[-1 if share[-1] else -2] += t - sum(lengths)
    return lengths
