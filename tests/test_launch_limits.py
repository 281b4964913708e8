"""Calls that one launch cannot hold and that are not split into several are refused on the host (fewer than 2^32 threads
along x; the runtime cuts a larger grid without an error)."""
import ctypes
import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, ROOT)
import sidekit_amd as sk        # noqa: E402

ARG, UNSUPPORTED = -1, -4
P = ctypes.c_void_p(0x1000)     # some address that is never followed


@pytest.fixture(scope="module")
def lib():
    return sk.load_library()


@pytest.fixture(scope="module")
def ctx():
    return ctypes.create_string_buffer(1024)        # no compute units, no profile


@pytest.mark.parametrize("M,N,K,rc", [(1, 0x7FFFFE00, 8, UNSUPPORTED), (16, 1 << 30, 512, UNSUPPORTED), (8, 1 << 27, 4096, UNSUPPORTED),
                                      (1 << 20, 1 << 20, 8, ARG)])
def test_product(lib, ctx, M, N, K, rc):
    assert lib.skm_gemm_fp8(ctx, P, P, 0, -1, 0, P, P, 0, M, N, K, P, 1, N, 0, None, 0, None) == rc


def test_experts_of_few_rows(lib, ctx):
    N = 0x7FFFFE00
    assert lib.skm_gemm_fp8_experts(ctx, P, P, 0, -1, 0, 4, P, P, 0, 4, N, 8, P, 2, 8, P, P, 16, P, P, P, 1, None, 0,
                                    None) == UNSUPPORTED


def test_tiles_and_columns(lib, ctx):
    wide = 0x7FFFFFFF
    assert lib.skm_fp8_tiles(ctx, P, 0, 1, 1, wide, wide, wide, 0, P, P, None, None, None) == ARG
    assert lib.skm_fp8_columns(ctx, P, 0, 8, wide, wide, 0, None, None, 0, None, 0, None, P, P, None) == ARG
