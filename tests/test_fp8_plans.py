"""Which kernel twm_gemm_fp8 runs, on the CPU: that every form is among the products that the GPU tests check, and that the
choice follows its rules."""
import ctypes as C

import pytest

import tensorwarp_amd as T
from tensorwarp_amd import _lib
from test_gpu_fp8 import GEMMS, LARGE_GEMMS


def form_of(m, n, k, dtype):
    parts = T.plan_fp8(m, n, k, dtype).split(", ")
    return parts[0] + ", " + parts[1] + ", " + parts[2] + (", split" if parts[3].endswith("splits") else "")


def test_every_form_is_tested_on_the_gpu():
    tested = {form_of(m, n, k, dtype) for m, n, k in GEMMS for dtype in ("f32", "f16")} | {form_of(*shape) for shape in LARGE_GEMMS}
    few = ["k_fp8_rows_few: %d columns x 16 rows, %d waves, f16 instructions" % v for v in ((16, 8), (16, 16), (32, 16), (32, 8), (16, 4))]
    few += ["k_fp8_rows_few: 32 columns x 16 rows, 8 waves, f16 instructions, split"]
    few += ["k_fp8_rows_few: %d columns x %d rows, 8 waves, f16 instructions%s" % (*form, split) for form in ((16, 32), (16, 64), (32, 64)) for split in ("", ", split")]
    tiles = ["k_fp8_tile: 128 columns x %d rows, 4 waves, %s instructions%s" % (rows, kind, split) for rows in (64, 128) for kind in ("8-bit", "f16")
             for split in ("", ", split")]
    tiles += ["k_fp8_tile: 256 columns x 256 rows, 8 waves, 8-bit instructions%s" % split for split in ("", ", split")]
    missing = [f for f in few + tiles if f not in tested]
    assert not missing, missing


@pytest.mark.parametrize("m", [1, 2, 15, 16])
def test_results_of_few_rows_come_from_exact_products(m):
    for n, k in ((1, 16), (896, 896), (4096, 11008), (11008, 4096), (37888, 3584)):
        for dtype in ("f32", "f16"):
            assert "k_fp8_rows_few" in T.plan_fp8(m, n, k, dtype) and "f16 instructions" in T.plan_fp8(m, n, k, dtype)


@pytest.mark.parametrize("m", [17, 100, 333, 2048])
def test_f32_results_come_from_exact_products(m):
    for n, k in ((1, 16), (896, 896), (4096, 11008), (37888, 3584)):
        assert "f16 instructions" in T.plan_fp8(m, n, k, "f32")


def test_splits_leave_every_range_blocks_and_fit_the_scratch():
    for m, n, k in ((17, 100, 18944), (64, 3584, 18944), (333, 3584, 18944), (2048, 256, 18944), (5000, 300, 1 << 20)):
        for dtype in ("f32", "f16"):
            splits = int(T.plan_fp8(m, n, k, dtype).split(", ")[-1].split()[0])
            blocks = -(-k // 128)
            per = -(-blocks // splits)
            assert (splits - 1) * per < blocks and splits * m * (n + 3) * 4 <= 256 << 20 or splits == 1


def test_describe_refusals():
    lib = _lib.load()
    buf = C.create_string_buffer(256)
    assert lib.twm_plan_describe_fp8(1, 64, 64, _lib.F32, None, 0) == _lib.INVALID_HANDLE
    assert lib.twm_plan_describe_fp8(1, 64, 60, _lib.F32, buf, 256) == _lib.SHAPE_ERROR
    assert lib.twm_plan_describe_fp8(1, 64, 64, _lib.U8, buf, 256) == _lib.UNSUPPORTED_OP
    assert T.plan_fp8(0, 64, 64) == "nothing to launch"
