"""The workspaces of the ops of a packed batch are no larger than the header says
(include/vx_hip_ops.h), over the extents that divide work."""

import re
from pathlib import Path

import pytest

from vx_amd.runtime import LIB_PATH, DispatchLibrary

HEADER = " ".join((Path(__file__).resolve().parent.parent / "include/vx_hip_ops.h").read_text().replace("*", " ").split())


@pytest.fixture(scope="module")
def lib():
    if not LIB_PATH.exists():
        from vx_amd.build import build
        build()
    return DispatchLibrary()


def test_gemm_i8(lib):
    most = int(re.search(r"the product (\d+) KiB a CU", HEADER).group(1)) * 1024 * 256
    assert f"{most >> 20} MiB on 256" in HEADER
    size, largest = lib.lib.vx_nn_gemm_i8_workspace, 0
    for tokens in (1, 16, 17, 31, 33, 48, 64, 65, 100, 128, 129, 200, 256, 500, 777, 1024, 2000, 4096):
        for rows in (1, 64, 100, 128, 512, 768, 1000, 1024, 2048, 4096, 6144, 11008, 32000):
            for cols in (16, 512, 768, 1024, 4096, 11008, 32768, 131056):
                n = size(tokens, rows, cols)
                assert 0 <= n <= most, (tokens, rows, cols, n)
                largest = max(largest, n)
    assert largest > most // 4  # the bound is near


def test_token_logprobs(lib):
    most = int(re.search(r"log probabilities use at most (\d+) KiB", HEADER).group(1)) * 1024
    size, largest = lib.lib.vx_nn_token_logprobs_workspace, 0
    for rows in [*range(1, 300), 512, 1000, 4096, 1 << 21]:
        for vocab in (1, 1000, 24575, 24576, 32000, 50257, 131072, 262144, 1 << 20, 1 << 30):
            for n_top in (0, 1, 5, 9, 20, 64):
                n = size(rows, vocab, n_top)
                assert 0 <= n <= most, (rows, vocab, n_top, n)
                largest = max(largest, n)
    assert largest > most // 2
