"""LDS blocks whose addresses kernels XOR: an address of a row XOR an offset in it
is the place meant only where rows begin on a multiple of their size, which the
declared alignment has to promise. As the compiler's front end declares it, before
anything is placed."""

import re
import subprocess

import pytest

from vx_amd.build import CSRC, HIP_FLAGS, hipcc


@pytest.mark.parametrize("source", ["flash_packed", "flash_shared"])
def test_rows_of_keys_begin_on_their_size(source, tmp_path):
    ir = tmp_path / f"{source}.ll"
    subprocess.run([hipcc(), *HIP_FLAGS, "--cuda-device-only", "-S", "-emit-llvm", "-Xclang", "-disable-llvm-passes",
                    str(CSRC / "kernels" / f"{source}.hip"), "-o", str(ir)], check=True, capture_output=True)
    blocks = re.findall(rf"^@\S*{source}ILi(\d+)E\S*3lds = internal addrspace\(3\) global \[\d+ x i8\] \w+, align (\d+)",
                        ir.read_text(), re.M)
    assert {int(d) for d, _ in blocks} == {64, 128}
    for head_dim, align in blocks:
        # a row: head_dim bf16
        assert int(align) % (2 * int(head_dim)) == 0, (head_dim, align)
