"""The choice of tiles, asked of the library without a GPU (CPU)."""

from __future__ import annotations

import ctypes
import subprocess
import sys

import pytest

import expert_tiles as et
from conftest import PACKAGE_DIR
from cuda_operator_lab import bindings as b
from test_abi import library


@pytest.fixture(scope="module", autouse=True)
def built():
    library()


@pytest.mark.parametrize("product,tiles,t,experts,n,k", et.CASES)
def test_each_case_runs_in_its_tiles(product, tiles, t, experts, n, k):
    assert b.expert_tiles(product, t, k, n, experts, et.SM_COUNT) == tiles
    lengths = et.ragged(t, experts)
    assert len(lengths) == experts and sum(lengths) == t and min(lengths) >= 0


def test_the_cases_cover_every_kernel():
    for product, kernels in et.KERNELS.items():
        assert {case[1] for case in et.CASES if case[0] == product} == kernels
    assert set(et.KERNELS) == set(b.EXPERT_PRODUCTS)


def test_no_size_chooses_tiles_without_a_kernel():
    sizes = (1, 2, 31, 33, 127, 129, 300, 1000, 4100, 16384, 200_000)
    for product, kernels in et.KERNELS.items():
        for t in sizes:
            for n in (128, 1024, 14336):
                for k in (16, 528, 4096):
                    for experts in ((1,) if product.startswith("dense") else (1, 7, 64, 1024)):
                        for sms in (2, 64, 132, et.SM_COUNT):
                            tiles = b.expert_tiles(product, t, k, n, experts, sms)
                            assert tiles in kernels, (product, t, n, k, experts, sms)


def test_rows_that_tma_cannot_address_are_the_cuda_cores():
    assert b.expert_tiles("bf16", 100, 1004, 64, 2, 148) is None
    assert b.expert_tiles("bf16", 100, 1000, 63, 2, 148) is not None
    for product in ("grad_input", "grad_weight", "both_grads"):
        assert b.expert_tiles(product, 100, 1000, 63, 2, 148) is None
        assert b.expert_tiles(product, 100, 1000, 64, 2, 148) is not None
    assert b.expert_tiles("fp8", 100, 1000, 64, 2, 148) is None
    assert b.expert_tiles("fp8", 100, 1008, 63, 2, 148) is not None


def test_refusals():
    call = b._library().handle.cuda_operator_lab_expert_tiles
    tiles = (ctypes.c_int * 4)()
    assert call(0, 1, 8, 8, 1, 148, tiles) == 0
    assert call(0, 1, 8, 8, 1, 148, None) == 1
    assert call(9, 1, 8, 8, 1, 148, tiles) == 1
    assert call(-1, 1, 8, 8, 1, 148, tiles) == 1
    assert call(7, 1, 16, 8, 2, 148, tiles) == 1  # a dense product has no experts
    for sizes in ((0, 8, 8, 1), (1, 0, 8, 1), (1, 8, 0, 1), (1, 8, 8, 0), (1 << 31, 8, 8, 1),
                  (1, 1 << 31, 8, 1), (1, 8, 1 << 31, 1), (1, 8, 8, 1025)):
        assert call(0, *sizes, 148, tiles) == 1, sizes
    assert call(0, 1, 8, 8, 1, 1, tiles) == 1
    with pytest.raises(ValueError):
        b.expert_tiles("no such product", 1, 8, 8, 1, 148)


def test_the_modules_import_under_a_torch_without_cuda():
    """Such a torch has no device query in its C module; calls are refused, not the import."""
    code = """
import sys, torch
del torch._C._cuda_getDevice
sys.path.insert(0, sys.argv[1])
from cuda_operator_lab import fp8, grouped
try:
    fp8.quantize_fp8_block128(torch.zeros(2, 128))
except ValueError as exc:
    assert "CUDA" in str(exc)
    print("refused")
"""
    done = subprocess.run([sys.executable, "-c", code, str(PACKAGE_DIR)], capture_output=True, text=True)
    assert done.returncode == 0 and "refused" in done.stdout, done.stderr
