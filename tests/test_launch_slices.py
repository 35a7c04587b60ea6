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


def test_slices_cover_the_rows_and_end_with_the_first_error(tmp_path):
    # (as the launchers do it: each launch's own error, nothing launched behind one that failed)
    body = """
    const unsigned cases[][3] = {{10, 4, 99}, {8, 4, 99}, {3, 4, 99}, {0, 4, 99}, {10, 4, 1}, {10, 4, 0}, {4294967295u, 2147483648u, 99}};
    for (auto &c : cases) {
        unsigned calls = 0;
        const int e = twm::in_slices(c[0], c[1], [&](unsigned row, unsigned count) { printf("%u+%u ", row, count); return calls++ == c[2] ? 7 : 0; });
        printf("= %d\\n", e);
    }"""
    assert run(tmp_path, body) == ["0+4 4+4 8+2 = 0", "0+4 4+4 = 0", "0+3 = 0", "= 0", "0+4 4+4 = 7", "0+4 = 7", "0+2147483648 2147483648+2147483647 = 0"]


def test_the_kernels_of_rows_are_launched_so():
    for name, launchers in (("twm_fp8_rows.hip", 2), ("twm_sample.hip", 1)):
        with open(os.path.join(build.CSRC, name)) as f:
            text = f.read()
        assert text.count("return in_slices(rows, most_workgroups(") == launchers and "row += " not in text
        # no launch whose error is not asked for before the next one
        launches = text.split("hipLaunchKernelGGL(")[1:]
        assert launches and all("hipGetLastError()" in after for after in launches), name
