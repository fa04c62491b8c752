"""Which plan attention over a shared prefix gets for the cases that the GPU
tests run (tests/test_gpu_flash_shared.py): every kernel, on its own and with
other workgroups, by either merge, is among them."""

import subprocess
from pathlib import Path

import pytest

from tests.test_gpu_flash_shared import CASES, PLANNED, SHORT

SRC = Path(__file__).resolve().parent / "native" / "shared_plan.cpp"


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    exe = tmp_path_factory.mktemp("plan") / "shared_plan"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", str(SRC), "-o", str(exe)], check=True)

    def of(cases):
        """(together, shared_rows, own_rows, tile, shared_splits, own_splits, parts) of each."""
        args = [str(x) for c in cases for x in c]
        out = subprocess.run([str(exe), *args], capture_output=True, text=True, check=True).stdout
        got = [tuple(map(int, line.split())) for line in out.splitlines()]
        assert len(got) == len(cases)
        return got

    return of


@pytest.mark.parametrize("head_dim", [64, 128])
def test_cases_are_divided_as_their_tests_say(plans, head_dim):
    table = [(c[0], c[-1]) for c in PLANNED + SHORT]
    for (ext, want), got in zip(table, plans([(*ext, head_dim) for ext, _ in table])):
        assert got[:6] == want, ext


@pytest.mark.parametrize("head_dim", [64, 128])
def test_every_plan_is_among_the_cases(plans, head_dim):
    """The kernel and what it walks; with and without divided own keys; merged
    by one thread a column and by four."""
    got = plans([(*c[0], head_dim) for c in PLANNED] + [c[:7] for c in CASES if c[6] == head_dim])
    kernels = {(1, 0, 1, 64), (1, 0, 0, 64), (1, 0, 0, 128),
               (0, 1, 1, 64), (0, 0, 1, 64), (0, 0, 1, 128), (0, 0, 0, 64), (0, 0, 0, 128)}
    assert {g[:4] for g in got} == kernels
    for which in (lambda g: g[5] == 1, lambda g: g[5] > 1, lambda g: 1 < g[6] <= 8, lambda g: g[6] > 8):
        assert {g[:4] for g in got if which(g)} == kernels
