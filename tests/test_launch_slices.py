"""How rows are shared out among launches, on the CPU: the header that says so has no device code and compiles by itself."""
import os
import shutil
import subprocess

import pytest

from tensorwarp_amd import build


def run(tmp_path, body):
    """What a program around twm_slices.h prints, line by line."""
    src = tmp_path / "slices.cpp"
    src.write_text('#include "twm_slices.h"\n#include <cstdio>\nint main()\n{\n%s\n}\n' % body)
    exe = str(tmp_path / "slices")
    subprocess.run([shutil.which("g++") or "c++", "-std=c++17", "-Wall", "-Werror", "-I", build.CSRC, str(src), "-o", exe], check=True)
    return subprocess.run([exe], check=True, stdout=subprocess.PIPE, text=True).stdout.split("\n")[:-1]


@pytest.mark.parametrize("threads", [128, 256, 1024])
def test_a_launch_has_fewer_than_2_to_the_32_threads(tmp_path, threads):
    # the workgroups of the norm's three forms, the gate's and the sampler's: 2^22 rows of 1024 threads are one launch too large
    most = int(run(tmp_path, 'printf("%%u\\n", twm::most_workgroups(%d));' % threads)[0])
    assert most * threads < 1 << 32 and most >= 1 << 21


def test_the_kernels_of_rows_take_their_limits_from_there():
    for name in ("twm_fp8_rows.hip", "twm_sample.hip"):
        with open(os.path.join(build.CSRC, name)) as f:
            text = f.read()
        loops = [line for line in text.split("\n") if "row += " in line]
        assert loops and all("row += most)" in line or "row += kMost)" in line for line in loops)
        assert text.count("most_workgroups(") == len(loops)
