"""The 8-bit floating point path -- rows with scales, their product with block-scaled weights -- and the token sampler, through
the C ABI, against plain numpy in 64 bits.

Tolerances count roundings.  e4m3 has three mantissa bits: a code is off by at most 2^-4 of its value, or 2^-10 where it is
subnormal.  Row functions compute y in f32 with no more than sixteen roundings of 2^-24: 2^-20 of y (and of gate * up, where
1 + tanh cancels).  A product of two e4m3 values is exact in f32; a block of 128 of them is added with at most 128 roundings (of
2^-23, should the matrix unit cut off instead of rounding), then comes one for the scales' product, one for the scaling and one
per addition of a block, a wave's or a K-range's sum.  Where results are f16 and rows are more than 16, the matrix unit may cut each
product of an aligned group of eight features off to a whole number of 2^(E - 13), E being the largest sum of the two codes'
exponents in the group (subnormal codes count as exponent -6): each product is off by less than that, eight together by less
than 2^-10 of 2^E."""
import numpy as np
import pytest

import tensorwarp_amd as T

pytestmark = pytest.mark.gpu

BLOCK = 128


@pytest.fixture(scope="module")
def dev():
    with T.WarpDevice(0) as d:
        yield d


def blocks(n):
    return -(-n // BLOCK)


def e4m3_table():
    t = np.zeros(256, np.float64)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        v = np.nan if e == 15 and m == 7 else m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        t[c] = -v if c & 128 else v
    return t


E4M3 = e4m3_table()


class Out:
    """An output buffer with sentinels on both sides, so that a store outside of it shows."""

    def __init__(self, dev, shape, dtype):
        self.n, self.shape, self.kind = int(np.prod(shape)), shape, dtype
        np_type = {"f32": np.float32, "f16": np.uint16, "u8": np.uint8, "i32": np.int32}[dtype]
        self.pad = 64
        self.fill = np.full(self.n + 2 * self.pad, 0x5A, np.uint8) if dtype == "u8" else np.full(self.n + 2 * self.pad, 12345, np_type)
        self.whole = T.GpuTensor.from_host(dev, self.fill, dtype)
        self.dtype, self.numel = dtype, self.n
        self.ptr = self.whole.ptr + self.pad * self.fill.itemsize

    def get(self):
        h = self.whole.to_host()
        assert np.array_equal(h[:self.pad], self.fill[:self.pad]) and np.array_equal(h[self.pad + self.n:], self.fill[self.pad + self.n:])
        v = h[self.pad:self.pad + self.n].reshape(self.shape)
        return v.view(np.float16) if self.kind == "f16" else v


class At:
    """A device array that begins `skip` elements into its allocation."""

    def __init__(self, dev, array, skip=0):
        flat = np.ascontiguousarray(array).reshape(-1)
        self.whole = T.GpuTensor.from_host(dev, np.concatenate([flat[:1].repeat(skip), flat]) if flat.size else np.zeros(16, flat.dtype))
        self.dtype = self.whole.dtype
        self.ptr = self.whole.ptr + skip * flat.itemsize


def check_codes(q, scales, y, y_err):
    """q, scales of rows y whose values are known within y_err (f64 arrays)."""
    rows, cols = y.shape
    kb = blocks(cols)
    for b in range(kb):
        at = slice(b * BLOCK, min((b + 1) * BLOCK, cols))
        amax, err = np.abs(y[:, at]).max(axis=1), y_err[:, at].max(axis=1)
        want = np.maximum(amax, 1e-30) / 448.0
        assert (np.abs(scales[:, b] - want) <= err / 448.0 + 2.0 ** -22 * want).all()
        s = scales[:, b].astype(np.float64)[:, None]
        v, off = y[:, at] / s, y_err[:, at] / s
        got = E4M3[q[:, at]]
        # half a step, the roundings of y * (448 / amax), and what y itself may be off
        assert (np.abs(got - v) <= np.maximum(2.0 ** -4 * np.abs(v), 2.0 ** -10) + 2.0 ** -21 * np.abs(v) + off).all()
        big = np.abs(got).max(axis=1)   # the block's largest is the largest code
        assert (big[amax > 1e-29] == 448.0).all()


SHAPES = [(1, 1), (1, 128), (3, 7), (2, 129), (1, 896), (5, 1000), (4, 2048), (3, 2049), (2, 4096), (2, 4104), (3, 5001), (2, 16392), (1, 50001)]


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantize_rows(dev, rows, cols, dtype):
    rng = np.random.default_rng(rows * 100003 + cols)
    x = (rng.standard_normal((rows, cols)) * np.exp(rng.uniform(-6, 4, (rows, 1)))).astype(np.float16 if dtype == "f16" else np.float32)
    x[:, :min(cols, 40)] *= (rng.random((rows, min(cols, 40))) > 0.5)   # some zeros
    q, s = Out(dev, (rows, cols), "u8"), Out(dev, (rows, blocks(cols)), "f32")
    T.quantize_rows_fp8(dev, At(dev, x), q, s, rows, cols)
    y = x.astype(np.float64)
    check_codes(q.get(), s.get(), y, np.zeros_like(y))


@pytest.mark.parametrize("skip", [1, 2, 4])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_rows_at_odd_addresses_are_the_aligned_rows(dev, dtype, skip):
    rng = np.random.default_rng(5)
    x = rng.standard_normal((3, 512)).astype(np.float16 if dtype == "f16" else np.float32)
    got = []
    for off in (0, skip):
        q, s = Out(dev, (3, 512), "u8"), Out(dev, (3, 4), "f32")
        T.quantize_rows_fp8(dev, At(dev, x, off), q, s, 3, 512)
        q2, s2 = Out(dev, (3, 256), "u8"), Out(dev, (3, 2), "f32")
        T.swiglu_rows_fp8(dev, At(dev, x, off), q2, s2, 256, 3)
        q3, s3, n3 = Out(dev, (3, 512), "u8"), Out(dev, (3, 4), "f32"), Out(dev, (3, 512), "f16")
        T.add_rms_norm_fp8(dev, At(dev, x, off), None, At(dev, np.ones(512, np.float32), off), 1e-6, 3, 512, q3, s3, normed=n3)
        got.append([t.get() for t in (q, s, q2, s2, q3, s3, n3)])
    for a, b in zip(*got):
        assert np.array_equal(a, b)


def test_blocks_of_zeros_tiny_values_infinities_and_nans(dev):
    x = np.zeros((1, 6 * BLOCK), np.float32)
    x[0, 128:256] = 1e-38
    x[0, 256 + 5] = np.inf
    x[0, 384 + 7] = np.nan
    x[0, 512:640] = 3.0e38
    x[0, 640:768] = -2.0
    q, s = Out(dev, x.shape, "u8"), Out(dev, (1, 6), "f32")
    T.quantize_rows_fp8(dev, At(dev, x), q, s, 1, x.shape[1])
    q, s = q.get()[0], s.get()[0]
    assert (q[:256] & 0x7F == 0).all() and (s[:2] > 0).all() and (s[:2] < 1e-30).all()
    assert np.isnan(s[2]) and np.isnan(s[3])
    assert (E4M3[q[512:640]] == 448.0).all() and abs(s[4] / (3.0e38 / 448) - 1) < 2.0 ** -22
    assert (E4M3[q[640:]] == -448.0).all() and abs(s[5] * 448 - 2.0) < 2.0 ** -22


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("rows,dim,paired", [(1, 1, 0), (3, 31, 0), (8, 704, 1), (2, 130, 0), (5, 1184, 1), (2, 4099, 0), (3, 2816, 0), (1, 32, 1), (33, 160, 1)])
def test_gated_rows(dev, rows, dim, paired, dtype, act):
    rng = np.random.default_rng(rows * 1009 + dim)
    x = (2.5 * rng.standard_normal((rows, 2 * dim))).astype(np.float16 if dtype == "f16" else np.float32)
    x[0, :2] = [-60.0, 60.0][:2]
    q, s = Out(dev, (rows, dim), "u8"), Out(dev, (rows, blocks(dim)), "f32")
    (T.swiglu_rows_fp8 if act == "silu" else T.geglu_rows_fp8)(dev, At(dev, x), q, s, dim, rows, paired=bool(paired))
    v = x.astype(np.float64)
    if paired:
        v = v.reshape(rows, dim // 32, 2, 32)
        g, u = v[:, :, 0].reshape(rows, dim), v[:, :, 1].reshape(rows, dim)
    else:
        g, u = v[:, :dim], v[:, dim:]
    y = g / (1 + np.exp(-g)) * u if act == "silu" else 0.5 * g * (1 + np.tanh(np.sqrt(2 / np.pi) * (g + 0.044715 * g ** 3))) * u
    check_codes(q.get(), s.get(), y, 2.0 ** -20 * (np.abs(y) + (np.abs(g * u) if act == "gelu" else 0)) + 1e-37)


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gates_whose_plain_product_no_f32_holds(dev, act):
    # act(g) is small enough for u, g u is not (e^-g is off by |g| roundings of 2^-24, act(g) by some more, for gelu |2 z| of them: 32 in all
    # at g = -5, where 2 z = 17)
    g = np.array([-20.0, -12.0, -3.0, 0.25] if act == "silu" else [-5.0, -3.0, -1.0, 0.25], np.float32)
    x = np.zeros((4, 64), np.float32)
    x[:, :32] = g[:, None]
    x[:, 32:] = np.float32(2.5e38) * np.linspace(-1, 1, 32).astype(np.float32)
    q, s = Out(dev, (4, 32), "u8"), Out(dev, (4, 1), "f32")
    (T.swiglu_rows_fp8 if act == "silu" else T.geglu_rows_fp8)(dev, At(dev, x), q, s, 32, 4)
    v, u = x[:, :32].astype(np.float64), x[:, 32:].astype(np.float64)
    y = v / (1 + np.exp(-v)) * u if act == "silu" else 0.5 * v * (1 + np.tanh(np.sqrt(2 / np.pi) * (v + 0.044715 * v ** 3))) * u
    check_codes(q.get(), s.get(), y, 2.0 ** -19 * np.abs(y))


@pytest.mark.parametrize("cols", [130, 1000, 4096, 9001])
def test_norm_of_rows_whose_squares_no_f32_holds(dev, cols):
    # without eps the norm of a row does not depend on its magnitude
    rng = np.random.default_rng(cols)
    x = (rng.standard_normal((6, cols)) * np.array([1e-36, 1e-30, 1e-21, 1e20, 1e30, 3e37])[:, None]).astype(np.float32)
    w = (1 + 0.3 * rng.standard_normal(cols)).astype(np.float32)
    q, s, n = Out(dev, (6, cols), "u8"), Out(dev, (6, blocks(cols)), "f32"), Out(dev, (6, cols), "f16")
    T.add_rms_norm_fp8(dev, At(dev, x), None, At(dev, w), 0.0, 6, cols, q, s, normed=n)
    v = x.astype(np.float64)
    y = v / np.sqrt((v * v).mean(axis=1, keepdims=True)) * w
    assert (np.abs(n.get().astype(np.float64) - y) <= (2.0 ** -11 + 2.0 ** -20) * np.abs(y) + 2.0 ** -25).all()
    check_codes(q.get(), s.get(), y, 2.0 ** -20 * np.abs(y))


@pytest.mark.parametrize("with_residual,with_sum,with_normed", [(1, 1, 1), (1, 0, 0), (0, 0, 1), (0, 1, 0)])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_add_rms_norm(dev, rows, cols, dtype, with_residual, with_sum, with_normed):
    rng = np.random.default_rng(rows * 7919 + cols)
    x = rng.standard_normal((rows, cols)).astype(np.float16 if dtype == "f16" else np.float32)
    r = (3 * rng.standard_normal((rows, cols))).astype(np.float32)
    w = (1 + 0.3 * rng.standard_normal(cols)).astype(np.float32)
    eps = 1e-5
    q, s = Out(dev, (rows, cols), "u8"), Out(dev, (rows, blocks(cols)), "f32")
    total = Out(dev, (rows, cols), "f32") if with_sum else None
    normed = Out(dev, (rows, cols), "f16") if with_normed else None
    T.add_rms_norm_fp8(dev, At(dev, x), At(dev, r) if with_residual else None, At(dev, w), eps, rows, cols, q, s, sum=total, normed=normed)
    v = x.astype(np.float32) + r if with_residual else x.astype(np.float32)
    if with_sum:
        assert np.array_equal(total.get(), v)
    v = v.astype(np.float64)
    y = v / np.sqrt((v * v).mean(axis=1, keepdims=True) + np.float64(np.float32(eps))) * w
    if with_normed:
        assert (np.abs(normed.get().astype(np.float64) - y) <= (2.0 ** -11 + 2.0 ** -20) * np.abs(y) + 2.0 ** -25).all()
    check_codes(q.get(), s.get(), y, 2.0 ** -20 * np.abs(y))


@pytest.mark.parametrize("cols", [512, 4096, 20000, 777])
def test_the_residual_is_updated_in_place(dev, cols):
    rng = np.random.default_rng(cols)
    x, r, w = (rng.standard_normal(s).astype(np.float32) for s in ((3, cols), (3, cols), (cols,)))
    q, s, apart = Out(dev, (3, cols), "u8"), Out(dev, (3, blocks(cols)), "f32"), Out(dev, (3, cols), "f32")
    T.add_rms_norm_fp8(dev, At(dev, x), At(dev, r), At(dev, w), 1e-6, 3, cols, q, s, sum=apart)
    q2, s2, same = Out(dev, (3, cols), "u8"), Out(dev, (3, blocks(cols)), "f32"), At(dev, r)
    T.add_rms_norm_fp8(dev, At(dev, x), same, At(dev, w), 1e-6, 3, cols, q2, s2, sum=same)
    assert np.array_equal(same.whole.to_host().reshape(3, cols), apart.get())
    assert np.array_equal(q.get(), q2.get()) and np.array_equal(s.get(), s2.get())


def test_more_rows_than_one_launch_takes(dev):
    rows = (1 << 22) + 77
    rng = np.random.default_rng(9)
    x = rng.standard_normal((rows, 1)).astype(np.float32)
    q, s, total = Out(dev, (rows, 1), "u8"), Out(dev, (rows, 1), "f32"), Out(dev, (rows, 1), "f32")
    T.add_rms_norm_fp8(dev, At(dev, x), At(dev, x), At(dev, np.array([0.5], np.float32)), 0.0, rows, 1, q, s, sum=total)
    assert np.array_equal(total.get(), x + x)
    # a row of one column is its own norm: 0.5 times its sign
    assert np.array_equal(E4M3[q.get()], np.sign(x) * 448.0) and (np.abs(s.get() * 448 - 0.5) < 2.0 ** -22).all()
    q, s = Out(dev, (rows, 1), "u8"), Out(dev, (rows, 1), "f32")
    T.quantize_rows_fp8(dev, At(dev, x), q, s, rows, 1)
    assert np.array_equal(E4M3[q.get()], np.sign(x) * 448.0) and (np.abs(s.get() * 448 - np.abs(x)) <= 2.0 ** -22 * np.abs(x)).all()


def test_a_norm_of_zeros_and_of_an_infinity(dev):
    x = np.zeros((3, 300), np.float32)
    x[1, 7] = np.inf
    x[2] = 1.0
    q, s, n = Out(dev, (3, 300), "u8"), Out(dev, (3, 3), "f32"), Out(dev, (3, 300), "f16")
    T.add_rms_norm_fp8(dev, At(dev, x), None, At(dev, np.ones(300, np.float32)), 0.0, 3, 300, q, s, normed=n)
    # 0 / sqrt(0 + 0) is no number; the rows beside are left alone
    assert np.isnan(s.get()[0]).all() and np.isnan(s.get()[1]).any()
    assert np.allclose(n.get()[2], 1.0) and (E4M3[q.get()[2]] == 448.0).all()
    q, s = Out(dev, (3, 300), "u8"), Out(dev, (3, 3), "f32")
    T.add_rms_norm_fp8(dev, At(dev, x), None, At(dev, np.ones(300, np.float32)), 1e-6, 3, 300, q, s)
    assert (q.get()[0] & 0x7F == 0).all() and np.isfinite(s.get()[0]).all()


# ---- products --------------------------------------------------------------------------------------------------------

def codes(rng, rows, cols):
    """Every code but the two NaNs, subnormal ones and zeros among them."""
    c = rng.integers(0, 254, (rows, cols), dtype=np.uint8)
    return c + (c >= 0x7F)


def gemm_truth(a, a_s, w, w_s):
    """(sum in 64 bits, sum of magnitudes)"""
    m, k = a.shape
    n = w.shape[0]
    af = E4M3[a] * np.repeat(a_s.astype(np.float64), BLOCK, axis=1)[:, :k]
    wf = E4M3[w] * np.repeat(np.repeat(w_s.astype(np.float64), BLOCK, axis=0)[:n], BLOCK, axis=1)[:, :k]
    return af @ wf.T, np.abs(af) @ np.abs(wf).T


def power(codes_):
    """The power of two of each code, as the matrix unit aligns products: 2^-6 for subnormal codes, zeros and up."""
    return 2.0 ** (np.maximum((codes_ >> 3) & 15, 1).astype(np.float64) - 7.0)


def cut_off(a, a_s, w, w_s):
    """Sum over the groups of eight features of 2^-10 times the group's largest power of two: what the 8-bit matrix instructions
    may be off by (zero codes take no part: their products are zero)."""
    m, k = a.shape
    n = w.shape[0]
    a_p, w_p = np.where(a & 0x7F, power(a), 0.0), np.where(w & 0x7F, power(w), 0.0)
    total = np.zeros((m, n))
    for g in range(0, k, 8):
        top = np.zeros((m, n))
        for i in range(g, g + 8):
            np.maximum(top, a_p[:, i, None] * w_p[None, :, i], out=top)
        b = g // BLOCK
        total += top * a_s[:, b, None] * np.repeat(w_s[:, b].astype(np.float64), BLOCK)[None, :n]
    return total * 2.0 ** -10


def gemm_inputs(rng, m, n, k):
    a, w = codes(rng, m, k), codes(rng, n, k)
    a_s = np.exp(rng.uniform(-6, -3, (m, blocks(k)))).astype(np.float32)
    w_s = np.exp(rng.uniform(-8, -5, (blocks(n), blocks(k)))).astype(np.float32)
    return a, a_s, w, w_s


def check_gemm(dev, inputs, m, n, k, dtype, skip=0):
    a, a_s, w, w_s = inputs
    c = Out(dev, (m, n), dtype)
    T.gemm_fp8(dev, At(dev, a), At(dev, a_s, skip), At(dev, w), At(dev, w_s, skip), m, n, k, c)
    got = c.get().astype(np.float64)
    truth, size = gemm_truth(*inputs)
    tol = (128 * 2.0 ** -23 + (blocks(k) + 32) * 2.0 ** -24) * size
    if dtype == "f16":
        if m > 16:
            tol += cut_off(*inputs)
        tol += 2.0 ** -11 * (np.abs(truth) + tol) + 2.0 ** -25
    worst = (np.abs(got - truth) - tol).max() if got.size else 0
    assert worst <= 0, worst
    return c


GEMMS = [(1, 1, 16), (1, 16, 128), (1, 17, 144), (2, 130, 272), (3, 64, 112), (1, 896, 896), (5, 256, 1024), (15, 129, 704), (16, 100, 2816), (17, 260, 640),
         (31, 384, 1040), (32, 128, 4096), (33, 1, 256), (40, 640, 704), (64, 300, 1152), (65, 96, 512), (77, 513, 384), (100, 255, 2064), (128, 512, 1024),
         (129, 257, 1040), (200, 384, 256), (256, 256, 128), (257, 640, 1296), (300, 1000, 528), (513, 130, 896), (1, 4096, 18944), (13, 4096, 4096), (7, 8, 16),
         (1030, 520, 272), (48, 3584, 2048), (17, 17, 6464), (30, 400, 8208), (50, 40, 3216), (70, 264, 4112), (70001, 5, 32), (1, 300001, 16), (3, 70000, 48),
         (33, 1401, 2064), (80, 2047, 256), (200, 850, 1040), (390, 333, 400), (450, 130, 1024), (450, 97, 400), (420, 260, 3216), (2, 4001, 5520), (7, 1001, 8208), (1, 130, 18944), (12, 2101, 10256), (16, 2050, 10240)]


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("m,n,k", GEMMS)
def test_gemm(dev, m, n, k, dtype):
    check_gemm(dev, gemm_inputs(np.random.default_rng(m * 31 + n * 17 + k), m, n, k), m, n, k, dtype, skip=(m + n) % 4)


# the forms that the planner keeps for larger products, at ragged sizes: 256 x 256 tiles, 128 x 128 ones, those with K-splits
LARGE_GEMMS = [(1500, 9000, 144, "f16"), (2049, 8200, 400, "f16"), (1500, 4100, 272, "f16"), (1500, 4100, 272, "f32"), (200, 9000, 4112, "f16"), (200, 9000, 4112, "f32"),
               (333, 3584, 18944, "f16"), (333, 3584, 18944, "f32"), (90, 5003, 2064, "f16"), (24, 3001, 9040, "f32"), (12, 20001, 1040, "f32"), (12, 20001, 4112, "f16"),
               (5, 9001, 1040, "f32"), (142, 11098, 5488, "f16"), (500, 24700, 272, "f16"), (1000, 24712, 400, "f16"),
               (520, 24697, 272, "f16"), (140, 12001, 6800, "f16"), (140, 12000, 6800, "f16"), (266, 19760, 400, "f32"), (137, 12001, 9040, "f16")]


@pytest.mark.parametrize("m,n,k,dtype", LARGE_GEMMS)
def test_gemm_large(dev, m, n, k, dtype):
    rng = np.random.default_rng(m * 31 + n * 17 + k)
    inputs = gemm_inputs(rng, m, n, k)
    c = Out(dev, (m, n), dtype)
    T.gemm_fp8(dev, *(At(dev, v) for v in inputs), m, n, k, c)
    got = c.get().astype(np.float64)
    # whole columns: the first and the last ones, those beside the tiles' borders, and some more
    some = np.unique(np.concatenate([np.arange(0, 40), np.arange(n - 40, n), np.arange(120, 136) % n, np.arange(248, 264) % n, rng.integers(0, n, 150)]))
    a, a_s, w, w_s = inputs
    part = (a, a_s, w[some], w_s)
    af = E4M3[a] * np.repeat(a_s.astype(np.float64), BLOCK, axis=1)[:, :k]
    wf = E4M3[w[some]] * np.repeat(w_s.astype(np.float64)[some // BLOCK], BLOCK, axis=1)[:, :k]
    truth, size = af @ wf.T, np.abs(af) @ np.abs(wf).T
    tol = (128 * 2.0 ** -23 + (blocks(k) + 32) * 2.0 ** -24) * size
    if dtype == "f16":
        if m > 16:   # (rows in turn, not all of them where there are thousands)
            rows = np.unique(np.concatenate([np.arange(0, m, max(1, m // 60)), np.arange(m - 8, m)]))
            truth, tol, got = truth[rows], tol[rows], got[rows]
            for g in range(0, k, 8):
                b = g // BLOCK
                ap, wp = (np.where(v & 0x7F, power(v), 0.0) for v in (a[rows, g:g + 8], part[2][:, g:g + 8]))
                tol += (ap[:, None, :] * wp[None]).max(axis=2) * a_s[rows, b, None] * w_s[some // BLOCK, b].astype(np.float64) * 2.0 ** -10
        tol += 2.0 ** -11 * (np.abs(truth) + tol) + 2.0 ** -25
    assert (np.abs(got[:, some] - truth) <= tol).all(), (np.abs(got[:, some] - truth) - tol).max()


def test_gemm_without_features_or_results(dev):
    one = At(dev, np.zeros(16, np.uint8))
    s = At(dev, np.ones(4, np.float32))
    for dtype in ("f32", "f16"):
        c = Out(dev, (3, 5), dtype)
        T.gemm_fp8(dev, one, s, one, s, 3, 5, 0, c)
        assert (c.get() == 0).all()
        c = Out(dev, (1, 1), dtype)
        T.gemm_fp8(dev, one, s, one, s, 0, 5, 16, c)
        T.gemm_fp8(dev, one, s, one, s, 5, 0, 16, c)
        assert c.whole.to_host()[c.pad] == 12345


@pytest.mark.parametrize("m", [1, 20, 70, 300])
def test_gemm_nan_rows_stay_in_their_row_and_column(dev, m):
    # a NaN code or a NaN scale reaches its own row or column and nothing else, also where K ends inside a block
    n, k = 200, 400
    a, a_s, w, w_s = gemm_inputs(np.random.default_rng(m), m, n, k)
    a[m - 1, 399] = 0x7F
    w[150, 3] = 0xFF
    c = Out(dev, (m, n), "f32")
    T.gemm_fp8(dev, At(dev, a), At(dev, a_s), At(dev, w), At(dev, w_s), m, n, k, c)
    got = np.isnan(c.get())
    want = np.zeros((m, n), bool)
    want[m - 1] = True
    want[:, 150] = True
    assert np.array_equal(got, want)


def test_gemm_is_the_same_every_time(dev):
    for m, n, k in ((1, 512, 8192), (24, 640, 4096), (200, 384, 4096)):
        inputs = [At(dev, v) for v in gemm_inputs(np.random.default_rng(m), m, n, k)]
        got = []
        for _ in range(3):
            c = Out(dev, (m, n), "f32")
            T.gemm_fp8(dev, *inputs, m, n, k, c)
            got.append(c.get())
        assert np.array_equal(got[0], got[1]) and np.array_equal(got[0], got[2])


# ---- sampling --------------------------------------------------------------------------------------------------------

def pick(x, u, temperature, top_k, top_p, min_p):
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    if x.size == 0 or np.all(x == -np.inf):
        return 0
    if not temperature > 0:
        return int(np.argmax(x))
    order = np.lexsort((np.arange(x.size), -x))
    order = order[x[order] > -np.inf]
    if top_k > 0:
        order = order[:top_k]
    top = x[order[0]]
    with np.errstate(invalid="ignore"):
        w = np.where(x[order] == top, 1.0, np.exp((x[order] - top) / float(temperature)))
    sums = np.cumsum(w)
    if not np.isnan(top_p):
        keep = max(1, int((sums - w < float(top_p) * sums[-1]).sum())) if top_p < 1 else w.size
        order, w = order[:keep], w[:keep]
    if not np.isnan(min_p):
        keep = w >= min(1.0, float(min_p))
        order, w = order[keep], w[keep]
    at = np.argsort(order)
    order, sums = order[at], np.cumsum(w[at])
    goal = 0.0 if not u > 0 else float(u) * sums[-1]
    found = np.nonzero(sums > goal)[0] if u < 1 or not u > 0 else []
    return int(order[found[0]]) if len(found) else int(order[np.nonzero(w[at] > 2.0 ** -38)[0][-1]])


def draw_tokens(dev, x, u, t=None, k=None, p=None, mp=None):
    rows, cols = x.shape
    as_f32 = lambda v: None if v is None else At(dev, np.asarray(v, np.float32))  # noqa: E731
    out = Out(dev, (rows,), "i32")
    T.sample(dev, At(dev, x), as_f32(u), out, rows, cols, temperature=as_f32(t), top_k=None if k is None else At(dev, np.asarray(k, np.int32)),
             top_p=as_f32(p), min_p=as_f32(mp))
    got = out.get()
    want = [pick(x[r], np.float32(u[r]), np.float32(1 if t is None else t[r]), 0 if k is None else int(k[r]), np.float32(np.nan if p is None else p[r]),
                 np.float32(np.nan if mp is None else mp[r])) for r in range(rows)]
    return got, np.asarray(want, np.int32)


@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 2), (5, 63), (4, 64), (9, 1000), (2, 1024), (3, 1025), (1, 4097), (17, 5000), (2, 16385), (6, 32000), (70, 8200),
                                       (1, 152064), (5, 151936), (300, 257), (90, 60000), (520, 2100)])
@pytest.mark.parametrize("spread", [0.3, 3.0])
def test_sample(dev, rows, cols, spread):
    rng = np.random.default_rng(rows * 13 + cols)
    x = (spread * rng.standard_normal((rows, cols))).astype(np.float32)
    u = rng.random(rows)
    assert np.array_equal(*draw_tokens(dev, x, u))
    t = rng.uniform(0.3, 1.5, rows)
    assert np.array_equal(*draw_tokens(dev, x, u, t))
    k = rng.integers(-1, 2 * cols if cols < 50 else 60, rows)
    assert np.array_equal(*draw_tokens(dev, x, u, t, k=k))
    assert np.array_equal(*draw_tokens(dev, x, u, t, p=rng.uniform(0.05, 1.0, rows)))
    assert np.array_equal(*draw_tokens(dev, x, u, t, mp=rng.uniform(0, 0.5, rows)))
    t[rng.random(rows) < 0.2] = 0
    assert np.array_equal(*draw_tokens(dev, x, u, t, k=rng.integers(1, cols + 1, rows), p=rng.uniform(0.5, 1.0, rows), mp=rng.uniform(0, 0.05, rows)))


@pytest.mark.parametrize("rows,cols", [(4, 900), (3, 40000), (2, 152064), (70, 32000)])
@pytest.mark.parametrize("spread", [1e-30, 1e-6, 0.003, 0.1])
def test_sample_among_close_logits(dev, rows, cols, spread):
    # thousands of tokens within a factor of e^(1/64); a row of equals, one that nothing but its first token sets apart, masks of the type's
    # lowest value, and temperatures that spread the row out again
    rng = np.random.default_rng(rows + cols)
    x = (spread * rng.standard_normal((rows, cols)) + (0.0 if spread < 1e-7 else 3.0)).astype(np.float32)
    x[0] = 0.7
    x[1, 1:] = x[1, 2]
    x[-1, ::3] = -np.inf
    x[-1, 1] = np.finfo(np.float32).min if rows > 3 else x[-1, 1]
    u = rng.random(rows)
    for t in (None, np.full(rows, 2.0), np.full(rows, spread), np.full(rows, spread / 30)):
        assert np.array_equal(*draw_tokens(dev, x, u, t, p=np.full(rows, 0.9)))
        assert np.array_equal(*draw_tokens(dev, x, u, t, k=rng.integers(1, cols + 1, rows), p=rng.uniform(0.1, 1.0, rows)))


@pytest.mark.parametrize("rows,cols", [(6, 1000), (5, 12288), (5, 12289), (3, 60000), (70, 40000)])
@pytest.mark.parametrize("most", [40, 100, 900])
def test_sample_by_both_limits(dev, rows, cols, most):
    # a small top_k's tokens are listed one and all, a large one's only where it ends; with few tokens that have any weight, and with many
    rng = np.random.default_rng(rows * 31 + cols + most)
    x = (2 * rng.standard_normal((rows, cols))).astype(np.float32)
    x[0, rng.permutation(cols)[:cols - 30]] = -1e9
    x[1, rng.permutation(cols)[:cols - 700]] = -np.inf
    x[2, rng.permutation(cols)[:300]] = 9.0
    u, t = rng.random(rows), rng.uniform(0.2, 1.5, rows)
    k, p = rng.integers(1, most + 1, rows), rng.uniform(0.3, 1.0, rows)
    for limits in (dict(k=k, p=p), dict(k=k), dict(k=np.full(rows, most), p=p), dict(k=k, p=np.ones(rows)), dict(k=k, p=np.full(rows, 1e-6)),
                   dict(k=k, p=p, mp=rng.uniform(0, 0.2, rows))):
        assert np.array_equal(*draw_tokens(dev, x, u, t, **limits))


@pytest.mark.parametrize("cols", [7, 1000, 40000])
def test_sample_among_equal_logits(dev, cols):
    # few distinct values, so that top-k and top-p end among equals, where the lower index stays
    rng = np.random.default_rng(cols)
    rows = 24
    x = rng.integers(0, 3, (rows, cols)).astype(np.float32) * np.float32(0.7)
    x[0] = 1.5
    x[1] = -0.0
    x[1, ::2] = 0.0
    u = rng.random(rows)
    k = rng.integers(1, cols + 1, rows)
    assert np.array_equal(*draw_tokens(dev, x, u, k=k))
    assert np.array_equal(*draw_tokens(dev, x, u, k=np.full(rows, 1)))
    assert np.array_equal(*draw_tokens(dev, x, u, mp=np.ones(rows)))
    # (sums of ones are exact: 3 of 8 of a row of equals)
    assert np.array_equal(*draw_tokens(dev, np.full((rows, cols), 2.5, np.float32), u, p=np.full(rows, 0.375)))
    assert np.array_equal(*draw_tokens(dev, x, u, t=np.zeros(rows)))


@pytest.mark.parametrize("cols", [50, 3000, 70000])
def test_sample_masks_and_numbers_that_are_none(dev, cols):
    rng = np.random.default_rng(cols)
    rows = 12
    x = (2 * rng.standard_normal((rows, cols))).astype(np.float32)
    x[0] = -np.inf                      # nothing allowed
    x[1] = np.nan
    x[2, :] = -np.inf
    x[2, cols - 1] = -5.0               # one token
    x[3, rng.random(cols) < 0.9] = -np.inf
    x[4, rng.random(cols) < 0.5] = np.nan
    x[5, [3, cols // 2]] = np.inf       # two that share the choice
    x[6] = np.finfo(np.float32).min     # a mask of the type's lowest value, over everything
    x[7, 5:] = np.finfo(np.float32).min
    x[8, cols // 3] = 3e38
    u = rng.random(rows)
    t = rng.uniform(0.5, 1.2, rows)
    for k, p, mp in ((None, None, None), (np.full(rows, 5), None, None), (None, np.full(rows, 0.9), None), (None, None, np.full(rows, 0.01)),
                     (np.full(rows, 40), np.full(rows, 0.8), np.full(rows, 0.02))):
        assert np.array_equal(*draw_tokens(dev, x, u, t, k=k, p=p, mp=mp))
        assert np.array_equal(*draw_tokens(dev, x, u, np.zeros(rows), k=k, p=p, mp=mp))


def test_sample_rules_at_their_ends(dev):
    rng = np.random.default_rng(8)
    x = rng.standard_normal((9, 300)).astype(np.float32)
    u = np.array([0.0, -1.0, np.nan, 1.0, 2.0, np.float32(1) - np.float32(2.0 ** -24), 0.5, 0.5, 0.5])
    assert np.array_equal(*draw_tokens(dev, x, u))
    some = rng.random(9)
    assert np.array_equal(*draw_tokens(dev, x, some, p=[0.0, -1.0, np.nan, 1.0, 2.0, 1e-30, 0.5, 0.999999, 0.1]))
    assert np.array_equal(*draw_tokens(dev, x, some, mp=[0.0, -1.0, np.nan, 1.0, 2.0, 1e-30, 0.5, 0.999999, 0.1]))
    assert np.array_equal(*draw_tokens(dev, x, some, t=[0.0, -1.0, np.nan, 1e-30, 1e30, np.inf, 1e-3, 50.0, -0.0]))
    assert np.array_equal(*draw_tokens(dev, x, some, k=[0, -5, 1, 2, 299, 300, 301, 2 ** 31 - 1, -2 ** 31]))


def test_sample_rows_without_columns(dev):
    out = Out(dev, (3,), "i32")
    T.sample(dev, At(dev, np.zeros(1, np.float32)), At(dev, np.zeros(3, np.float32)), out, 3, 0)
    assert np.array_equal(out.get(), [0, 0, 0])


def test_sample_more_rows_than_one_launch_takes(dev):
    rows = (1 << 21) + 5
    rng = np.random.default_rng(10)
    x = rng.standard_normal((rows, 2)).astype(np.float32)
    u = rng.random(rows).astype(np.float32)
    out = Out(dev, (rows,), "i32")
    T.sample(dev, At(dev, x), At(dev, u), out, rows, 2)
    p0 = 1.0 / (1.0 + np.exp(x[:, 1].astype(np.float64) - x[:, 0]))
    clear = np.abs(p0 - u) > 1e-9   # (nearer than that, two roundings of 2^-50 could decide)
    assert clear.sum() > rows - 10 and np.array_equal(out.get()[clear], (u >= p0)[clear].astype(np.int32))


def test_sampling_leaves_the_counters_that_others_share_at_zero(dev):
    # arrival counters belong to the context: argmax over several spans and the few-row sampler in turn, twice
    rng = np.random.default_rng(6)
    x = (2 * rng.standard_normal((5, 60000))).astype(np.float32)
    xd, top = At(dev, x), Out(dev, (5,), "i32")
    for _ in range(2):
        assert np.array_equal(*draw_tokens(dev, x, rng.random(5), p=np.full(5, 0.9)))
        T.argmax(dev, xd, top, 5, 60000)
        assert np.array_equal(top.get(), np.argmax(x, axis=1))
        assert np.array_equal(*draw_tokens(dev, x, rng.random(5), k=np.full(5, 30)))


def test_two_captured_graphs_that_share_the_scratch(dev):
    # a product with K-splits and a sampler of few rows each park sums in the context's scratch; replayed in turn, with other work
    # between, both give what the eager calls give
    rng = np.random.default_rng(12)
    m, n, k = 20, 500, 9088
    assert "splits" in T.plan_fp8(m, n, k)
    inputs = [At(dev, v) for v in gemm_inputs(rng, m, n, k)]
    logits, u = At(dev, (2 * rng.standard_normal((3, 50000))).astype(np.float32)), At(dev, rng.random(3).astype(np.float32))
    p = At(dev, np.full(3, 0.9, np.float32))
    c, token = Out(dev, (m, n), "f32"), Out(dev, (3,), "i32")
    calls = [lambda: T.gemm_fp8(dev, *inputs, m, n, k, c), lambda: T.sample(dev, logits, u, token, 3, 50000, top_p=p)]
    for call in calls:
        call()
    want = c.get(), token.get()
    graphs = [T.GraphCapture.record_with_device(dev, call) for call in calls]
    for order in ((0, 1), (1, 0), (0, 0, 1, 1), (1, 0, 1)):
        c.whole.copy_from_host(c.fill)
        token.whole.copy_from_host(token.fill)
        for i in order:
            graphs[i].replay()
        assert np.array_equal(c.get(), want[0]) and np.array_equal(token.get(), want[1])
        calls[order[0]]()
    for g in graphs:
        g.destroy()


def test_a_rows_token_does_not_depend_on_the_batch(dev):
    rng = np.random.default_rng(4)
    x = (2 * rng.standard_normal((80, 9000))).astype(np.float32)
    u, p = rng.random(80), np.full(80, 0.95)
    together, _ = draw_tokens(dev, x, u, p=p)
    for r in (0, 41, 79):
        alone, _ = draw_tokens(dev, x[r:r + 1], u[r:r + 1], p=p[:1])
        assert alone[0] == together[r]


# ---- arrays beyond 4 GB ------------------------------------------------------------------------------------------------

class Big:
    """Zeros in device memory that are written and read in places."""

    def __init__(self, dev, nbytes):
        self.dev, self.lib, nbytes = dev, T._lib.load(), (nbytes + 3) // 4 * 4
        self.ptr = self.lib.twm_malloc(dev.handle, nbytes)
        assert self.ptr, self.lib.twm_last_error()
        self.nbytes = nbytes
        T.quantize._check(self.lib.twm_memset_zero(dev.handle, self.ptr, nbytes))

    def put(self, at, array):
        array = np.ascontiguousarray(array)
        assert at + array.nbytes <= self.nbytes
        T.quantize._check(self.lib.twm_memcpy_h2d(self.dev.handle, self.ptr + at, array.ctypes.data, array.nbytes))

    def take(self, at, count, dtype):
        out = np.empty(count, dtype)
        assert at + out.nbytes <= self.nbytes
        T.quantize._check(self.lib.twm_memcpy_d2h(self.dev.handle, out.ctypes.data, self.ptr + at, out.nbytes))
        return out

    def free(self):
        self.lib.twm_free(self.dev.handle, self.ptr)


@pytest.mark.parametrize("m,dtype", [(1, "f32"), (20, "f32"), (150, "f16"), (150, "f32")])
def test_gemm_with_weights_beyond_4_gb(dev, m, dtype):
    n, k, some = 270001, 16400, 300
    a, a_s, w, w_s = gemm_inputs(np.random.default_rng(m), m, some + BLOCK, k)
    first = (n - some) // BLOCK * BLOCK   # the last columns are not zeros: their rows' blocks begin here
    w, w_s = w[:n - first], np.exp(np.random.default_rng(1).uniform(-8, -5, (blocks(n), blocks(k)))).astype(np.float32)
    weights, c = Big(dev, n * k + 16), Big(dev, m * n * 4 + 16)
    weights.put(first * k, w)
    out = At(dev, np.zeros(1, np.float32))
    out.ptr, out.dtype = c.ptr, dtype
    rows = At(dev, w)
    rows.ptr = weights.ptr
    T.gemm_fp8(dev, At(dev, a), At(dev, a_s), rows, At(dev, w_s), m, n, k, out)
    got = c.take(0, m * n, np.float32 if dtype == "f32" else np.float16).reshape(m, n).astype(np.float64)
    assert (got[:, :first] == 0).all()
    inputs = a, a_s, w, w_s[first // BLOCK:]
    truth, size = gemm_truth(*inputs)
    tol = (128 * 2.0 ** -23 + (blocks(k) + 32) * 2.0 ** -24) * size
    if dtype == "f16":
        tol += cut_off(*inputs)
        tol += 2.0 ** -11 * (np.abs(truth) + tol) + 2.0 ** -25
    assert (np.abs(got[:, first:] - truth) <= tol).all()
    weights.free()
    c.free()


def test_rows_beyond_4_gb(dev):
    rows, cols = 1050001, 4104
    x, q, s = Big(dev, rows * cols * 2), Big(dev, rows * cols + 3), Big(dev, rows * blocks(cols) * 4)
    last = np.random.default_rng(2).standard_normal((2, cols)).astype(np.float16)
    x.put((rows - 2) * cols * 2, last)
    as_array = lambda big, dtype: type("Rows", (), {"ptr": big.ptr, "dtype": dtype})  # noqa: E731
    one = At(dev, np.ones(cols, np.float32))
    for norm in (False, True):
        if norm:
            T.add_rms_norm_fp8(dev, as_array(x, "f16"), None, one, 1e-6, rows, cols, as_array(q, "u8"), as_array(s, "f32"))
        else:
            T.quantize_rows_fp8(dev, as_array(x, "f16"), as_array(q, "u8"), as_array(s, "f32"), rows, cols)
        y = last.astype(np.float64)
        y = y / np.sqrt((y * y).mean(axis=1, keepdims=True) + 1e-6) if norm else y
        codes_, scales = q.take((rows - 2) * cols, 2 * cols, np.uint8), s.take((rows - 2) * blocks(cols) * 4, 2 * blocks(cols), np.float32)
        check_codes(codes_.reshape(2, cols), scales.reshape(2, -1), y, 2.0 ** -20 * np.abs(y))
        assert (q.take((rows - 3) * cols, cols, np.uint8) == 0).all()
    # (as a gate's rows: two of 2 * 2052 columns)
    T.swiglu_rows_fp8(dev, as_array(x, "f16"), as_array(q, "u8"), as_array(s, "f32"), cols // 2, rows)
    g, u = last.astype(np.float64)[:, :cols // 2], last.astype(np.float64)[:, cols // 2:]
    y = g / (1 + np.exp(-g)) * u
    kb = blocks(cols // 2)
    codes_, scales = q.take((rows - 2) * (cols // 2), cols, np.uint8), s.take((rows - 2) * kb * 4, 2 * kb, np.float32)
    check_codes(codes_.reshape(2, -1), scales.reshape(2, -1), y, 2.0 ** -20 * np.abs(y) + 1e-37)
    for big in (x, q, s):
        big.free()


def test_sample_logits_beyond_4_gb(dev):
    rows, cols = 20000, 65540
    x = Big(dev, rows * cols * 4)
    last = (3 * np.random.default_rng(3).standard_normal((1, cols))).astype(np.float32)
    x.put((rows - 1) * cols * 4, last)
    t = np.zeros(rows, np.float32)
    t[-1] = 0.8
    u = np.full(rows, 0.6, np.float32)
    out = Out(dev, (rows,), "i32")
    T.sample(dev, type("Rows", (), {"ptr": x.ptr, "dtype": "f32"}), At(dev, u), out, rows, cols, temperature=At(dev, t))
    got = out.get()
    assert (got[:-1] == 0).all() and got[-1] == pick(last[0], u[-1], t[-1], 0, np.float32(np.nan), np.float32(np.nan))
    x.free()


# ---- the run of them, as a decode step makes it ------------------------------------------------------------------------

class Step:
    """A feed-forward block and the vocabulary's projection for m tokens: norm, gate and up, gate, down, norm, logits, token."""

    def __init__(self, dev, m, hidden, ffn, vocab, seed):
        rng = np.random.default_rng(seed)
        self.dev, self.m, self.hidden, self.ffn, self.vocab = dev, m, hidden, ffn, vocab
        self.h_w = {name: (codes(rng, n, k) & 0xBF, np.exp(rng.uniform(-4, -3, (blocks(n), blocks(k)))).astype(np.float32))
                    for name, n, k in (("gate_up", 2 * ffn, hidden), ("down", hidden, ffn), ("head", vocab, hidden))}
        self.w = {name: (At(dev, c), At(dev, s)) for name, (c, s) in self.h_w.items()}
        self.h_norms = [(1 + 0.1 * rng.standard_normal(hidden)).astype(np.float32) for _ in range(2)]
        self.norms = [At(dev, v) for v in self.h_norms]
        self.x, self.residual, self.uniform = (T.GpuTensor(dev, s, "f32") for s in ((m, hidden), (m, hidden), (m,)))
        self.stream_rows = T.GpuTensor(dev, (m, hidden), "f32")
        self.out = {"sum": Out(dev, (m, hidden), "f32"), "q1": Out(dev, (m, hidden), "u8"), "s1": Out(dev, (m, blocks(hidden)), "f32"),
                    "gate_up": Out(dev, (m, 2 * ffn), "f16"), "q2": Out(dev, (m, ffn), "u8"), "s2": Out(dev, (m, blocks(ffn)), "f32"),
                    "down": Out(dev, (m, hidden), "f32"), "sum2": Out(dev, (m, hidden), "f32"), "q3": Out(dev, (m, hidden), "u8"),
                    "s3": Out(dev, (m, blocks(hidden)), "f32"), "logits": Out(dev, (m, vocab), "f32"), "token": Out(dev, (m,), "i32")}
        self.k, self.p = At(dev, np.full(m, 50, np.int32)), At(dev, np.full(m, 0.95, np.float32))

    def give(self, seed):
        rng = np.random.default_rng(seed)
        self.h_x, self.h_residual = (rng.standard_normal((self.m, self.hidden)).astype(np.float32) for _ in range(2))
        self.h_uniform = rng.random(self.m).astype(np.float32)
        self.x.copy_from_host(self.h_x)
        self.residual.copy_from_host(self.h_residual)
        self.uniform.copy_from_host(self.h_uniform)

    def run(self):
        o, m, h, f, v, dev = self.out, self.m, self.hidden, self.ffn, self.vocab, self.dev
        T.add_rms_norm_fp8(dev, self.x, self.residual, self.norms[0], 1e-6, m, h, o["q1"], o["s1"], sum=o["sum"])
        T.gemm_fp8(dev, o["q1"], o["s1"], *self.w["gate_up"], m, 2 * f, h, o["gate_up"])
        T.swiglu_rows_fp8(dev, o["gate_up"], o["q2"], o["s2"], f, m)
        T.gemm_fp8(dev, o["q2"], o["s2"], *self.w["down"], m, h, f, o["down"])
        T.add_rms_norm_fp8(dev, o["down"], o["sum"], self.norms[1], 1e-6, m, h, o["q3"], o["s3"], sum=o["sum2"])
        T.gemm_fp8(dev, o["q3"], o["s3"], *self.w["head"], m, v, h, o["logits"])
        T.sample(dev, o["logits"], self.uniform, o["token"], m, v, top_k=self.k, top_p=self.p)

    def got(self):
        return {name: t.get() for name, t in self.out.items()}

    def check(self, g):
        """Every stage against 64 bits, from what the stage before it left."""
        def rows_of(x, w):
            v = x.astype(np.float64)
            return v / np.sqrt((v * v).mean(axis=1, keepdims=True) + 1e-6) * w
        assert np.array_equal(g["sum"], self.h_x + self.h_residual) and np.array_equal(g["sum2"], g["down"] + g["sum"])
        for q, s, total, w in (("q1", "s1", "sum", self.h_norms[0]), ("q3", "s3", "sum2", self.h_norms[1])):
            y = rows_of(g[total], w)
            check_codes(g[q], g[s], y, 2.0 ** -20 * np.abs(y))
        for q, s, w, c, k in (("q1", "s1", "gate_up", "gate_up", self.hidden), ("q2", "s2", "down", "down", self.ffn), ("q3", "s3", "head", "logits", self.hidden)):
            truth, size = gemm_truth(g[q], g[s], *self.h_w[w])
            tol = (128 * 2.0 ** -23 + (blocks(k) + 32) * 2.0 ** -24) * size
            if c == "gate_up":
                if self.m > 16:
                    tol += cut_off(g[q], g[s], *self.h_w[w])
                tol += 2.0 ** -11 * (np.abs(truth) + tol) + 2.0 ** -25
            assert (np.abs(g[c].astype(np.float64) - truth) <= tol).all(), c
        gu = g["gate_up"].astype(np.float64)
        gate, up = gu[:, :self.ffn], gu[:, self.ffn:]
        y = gate / (1 + np.exp(-gate)) * up
        check_codes(g["q2"], g["s2"], y, 2.0 ** -20 * np.abs(y) + 1e-37)
        want = [pick(g["logits"][r], self.h_uniform[r], np.float32(1), 50, np.float32(0.95), np.float32(np.nan)) for r in range(self.m)]
        assert np.array_equal(g["token"], want)


@pytest.mark.parametrize("m,hidden,ffn,vocab", [(1, 256, 704, 5000), (7, 384, 512, 2001), (140, 256, 640, 1000)])
def test_a_step_eager_captured_and_on_another_stream(dev, m, hidden, ffn, vocab):
    step = Step(dev, m, hidden, ffn, vocab, m)
    step.give(1)
    step.run()
    first = step.got()
    step.check(first)
    graph = T.GraphCapture.record_with_device(dev, step.run)
    for seed in (2, 1, 3):
        step.give(seed)
        graph.replay()
        dev.synchronize()
        replayed = step.got()
        step.run()   # eager work between the replays
        dev.synchronize()
        eager = step.got()
        assert all(np.array_equal(replayed[name], eager[name], equal_nan=True) for name in eager)
        step.check(eager)
    graph.destroy()
    lib = T._lib.load()
    stream = lib.twm_stream_create(dev.handle)
    dev.with_stream(stream)
    step.give(1)
    step.run()
    again = step.got()
    dev.with_stream(None)
    assert lib.twm_stream_destroy(dev.handle, stream) == T._lib.OK
    assert all(np.array_equal(first[name], again[name]) for name in first)
