"""What include/twmarlin.h says of the 8-bit path to the last bit, and its kernels where they are least at ease, through the C ABI
against plain numpy."""
import numpy as np
import pytest

import tensorwarp_amd as T
from test_gpu_fp8 import BLOCK, E4M3, At, Big, Out, blocks, check_codes

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    with T.WarpDevice(0) as d:
        yield d


def nearest_codes(v):
    """f32 values of at most 448 and a rounding as e4m3, ties to the even code."""
    table, m = E4M3[:0x7F], np.abs(v.astype(np.float64))
    lo = np.clip(np.searchsorted(table, m, side="right") - 1, 0, 0x7D)
    border = (table[lo] + table[lo + 1]) / 2
    code = lo + ((m > border) | ((m == border) & (lo % 2 == 1)))
    return (code | np.signbit(v) * 0x80).astype(np.uint8)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("rows,cols", [(300, 4096), (2000, 1000), (40, 11007)])
def test_codes_are_the_nearest_to_the_quotient_with_the_stored_scale(dev, rows, cols, dtype):
    # x / scale in f32 and from there the nearest code, to the bit: a division, not a product with an inverse rounded on its own
    rng = np.random.default_rng(rows + cols)
    x = rng.standard_normal((rows, cols)) * np.exp(rng.uniform(-3, 3, (rows, 1)))
    if dtype == "f32":
        x[::7] *= 10.0 ** rng.uniform(-29, -20, (len(x[::7]), 1))   # (blocks down to where the least scale begins)
        x[1::7] *= 10.0 ** rng.uniform(20, 36, (len(x[1::7]), 1))
    x = x.astype(np.float16 if dtype == "f16" else np.float32)
    q, s = Out(dev, (rows, cols), "u8"), Out(dev, (rows, blocks(cols)), "f32")
    T.quantize_rows_fp8(dev, At(dev, x), q, s, rows, cols)
    x, q, s = x.astype(np.float32), q.get(), s.get()
    padded = np.zeros((rows, blocks(cols) * BLOCK), np.float32)
    padded[:, :cols] = np.abs(x)
    amax = np.maximum(padded.reshape(rows, -1, BLOCK).max(axis=2), np.float32(1e-30))
    assert np.array_equal(s, amax / np.float32(448))
    want = nearest_codes(x / np.repeat(s, BLOCK, axis=1)[:, :cols])
    assert np.array_equal(q, want), (q != want).sum()


def test_norm_of_more_wide_rows_than_one_launch_takes(dev):
    # rows of more than 4096 columns take 1024 threads each: 2^22 rows are two launches of 2^31 threads, and three more rows a third
    rows, cols, at = (1 << 22) + 3, 4104, [0, (1 << 21) - 1, 1 << 21, (1 << 22) - 1, 1 << 22, (1 << 22) + 2]
    x, q, s = Big(dev, rows * cols * 2), Big(dev, rows * cols), Big(dev, rows * blocks(cols) * 4)
    some = np.random.default_rng(31).standard_normal((len(at), cols)).astype(np.float16)
    for r, v in zip(at, some):
        x.put(r * cols * 2, v)
    as_array = lambda big, dtype: type("Rows", (), {"ptr": big.ptr, "dtype": dtype})  # noqa: E731
    T.add_rms_norm_fp8(dev, as_array(x, "f16"), None, At(dev, np.ones(cols, np.float32)), 1e-6, rows, cols, as_array(q, "u8"), as_array(s, "f32"))
    y = some.astype(np.float64)
    y = y / np.sqrt((y * y).mean(axis=1, keepdims=True) + 1e-6)
    codes_ = np.stack([q.take(r * cols, cols, np.uint8) for r in at])
    scales = np.stack([s.take(r * blocks(cols) * 4, blocks(cols), np.float32) for r in at])
    check_codes(codes_, scales, y, 2.0 ** -20 * np.abs(y))
    for r in (1, (1 << 21) + 1, (1 << 22) + 1):   # (rows of zeros beside them)
        assert (q.take(r * cols, cols, np.uint8) == 0).all() and (s.take(r * blocks(cols) * 4, blocks(cols), np.float32) > 0).all()
    for big in (x, q, s):
        big.free()
