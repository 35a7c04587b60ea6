"""The quotient from which the row kernels take their codes, on the CPU: the header that holds it has no device code, and here it
falls on the side of every border between two codes on which the division's own falls."""
import shutil
import subprocess

from tensorwarp_amd import build

PROGRAM = r"""
#include "twm_e4m3.h"
#include <cstdint>
#include <cstdio>
#include <cstring>
static float from(uint32_t u) { float f; memcpy(&f, &u, 4); return f; }
static uint32_t bits(float f) { uint32_t u; memcpy(&u, &f, 4); return u; }
int main()
{
    float border[126];
    double before = 0;
    for (int c = 1; c < 127; c++) {
        const int e = c >> 3, m = c & 7;
        const double v = e ? (8 + m) * (e < 10 ? 1.0 / (1 << (10 - e)) : (double)(1 << (e - 10))) : m / 512.0;
        border[c - 1] = (float)((v + before) / 2);
        before = v;
    }
    long long off = 0, off_alone = 0, all = 0;
    // every STEP-th mantissa of a block's largest magnitude, for the least scales that take this way, ordinary and the largest ones
    const int exponents[] = {-81, -60, 0, 3, 127};
    for (int e : exponents)
        for (uint32_t m = (uint32_t)(e + 81); m < 1u << 23; m += 251) {
            const float amax = from((uint32_t)(e + 127) << 23 | m), scale = amax / twm::kFp8Max, inverse = twm::kFp8Max / amax;
            if (scale < twm::kFp8LeastExact) continue;
            for (float b : border)
                for (int d = -2; d <= 2; d++) {
                    const float x = from(bits((float)((double)scale * b)) + d), q = x / scale, u = twm::units_of(x, scale, inverse), alone = x * inverse;
                    off += (q > b) != (u > b) || (q < b) != (u < b);
                    off_alone += (q > b) != (alone > b) || (q < b) != (alone < b);
                    all++;
                }
        }
    printf("%lld %lld %lld\n", off, off_alone, all);
}
"""


def test_units_fall_on_the_quotients_side_of_every_border(tmp_path):
    src, exe = tmp_path / "codes.cpp", str(tmp_path / "codes")
    src.write_text(PROGRAM)
    subprocess.run([shutil.which("g++") or "c++", "-std=c++17", "-O2", "-ffp-contract=off", "-Wall", "-Werror", "-I", build.CSRC, str(src), "-o", exe], check=True)
    off, off_alone, count = (int(v) for v in subprocess.run([exe], check=True, stdout=subprocess.PIPE, text=True).stdout.split())
    assert count > 7e7 and off == 0
    assert off_alone > count / 10   # (what the remainder's step is for)
