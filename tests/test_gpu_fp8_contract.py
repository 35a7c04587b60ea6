"""What include/twmarlin.h says of the 8-bit path to the last bit, and its kernels where they are least at ease, through the C ABI
against plain numpy."""
import numpy as np
import pytest

import tensorwarp_amd as T
from test_gpu_fp8 import BLOCK, E4M3, At, Big, Out, blocks, check_codes, draw_tokens, gemm_inputs

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


def gates(act, g, u):
    """act(g) * u in 64 bits, without a difference of nearly equal numbers and without an overflow on the way."""
    g, u = g.astype(np.float64), u.astype(np.float64)
    z2 = g if act == "silu" else 2 * np.sqrt(2 / np.pi) * (g + 0.044715 * g ** 3)
    e = np.exp(-np.abs(z2))
    return g * u * np.where(z2 > 0, 1.0, e) / (1 + e)


def gate_of_single_columns(dev, act, g, u):
    """|y| as the scales of rows of one column have it, and the codes."""
    rows = len(g)
    x = np.stack([g, u], axis=1)
    q, s = Out(dev, (rows, 1), "u8"), Out(dev, (rows, 1), "f32")
    (T.swiglu_rows_fp8 if act == "silu" else T.geglu_rows_fp8)(dev, At(dev, x), q, s, 1, rows)
    return s.get()[:, 0].astype(np.float64) * 448, q.get()[:, 0]


def gate_error(act, g):
    """An exponential and a reciprocal of an ulp each, 2^-23, and four roundings of 2^-24 -- 1 + e, act(g), times u, the exponential's
    low part -- are 2^-21 of y; the scale's division rounds by 2^-24 again.  gelu's exponent is g (c + d g^2): half an ulp of g^2 and of
    the bracket, and what f32 leaves of c and d, make as much of e^2z as they are of 2z's logarithm to base two, times ln 2."""
    error = np.full(g.shape, 2.0 ** -21 + 2.0 ** -24)
    if act == "gelu":
        c = 2 * np.sqrt(2 / np.pi) * np.log2(np.e)
        d, square = 0.044715 * c, np.minimum(g.astype(np.float64) ** 2, 1e4)   # (from g = 100 on 1 + e is one)
        half = lambda v: np.spacing(v.astype(np.float32)).astype(np.float64) / 2  # noqa: E731
        bracket = half(c + d * square) + d * half(square) + square * abs(d - float(np.float32(d))) + abs(c - float(np.float32(c)))
        error += np.log(2) * np.minimum(np.abs(g), 100.0) * bracket * 1.001
    return error


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gates_are_as_near_as_their_roundings(dev, act):
    # relative to the gate itself, also where it is far below zero and its exponent's roundings count most
    rng = np.random.default_rng(21)
    g = np.concatenate([rng.uniform(-9, 9, 200000), rng.uniform(-80, -9, 20000) if act == "silu" else rng.uniform(-8.9, -3, 20000),
                        10.0 ** rng.uniform(-20, 0, 20000), -10.0 ** rng.uniform(-20, 0, 20000), 10.0 ** rng.uniform(1, 15, 2000)]).astype(np.float32)
    u = rng.uniform(0.5, 2.0, len(g)).astype(np.float32) * np.where(g < -30, np.float32(1e20), np.float32(1))
    y = gates(act, g, u)
    seen = np.abs(y) > 1e-29
    assert seen.sum() > len(g) - 100
    got, codes_ = gate_of_single_columns(dev, act, g, u)
    off = (np.abs(got - np.abs(y)) / np.abs(y) / gate_error(act, g))[seen]
    assert off.max() <= 1, (off.max(), g[seen][off.argmax()])
    assert np.array_equal(codes_[seen] >> 7, y[seen] < 0)


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gates_that_vanish(dev, act):
    # act(g) falls off like e^g beyond what f32 holds: with a large u it still is a number of its own there, and with any other u it
    # is nothing, not a floor that stays in a block of small values
    rng = np.random.default_rng(22)
    least = (-260.0, -20.0)[act == "gelu"]
    g = np.concatenate([rng.uniform(least, least / 3, 60000), [-1e3, -1e6, -3e38] * 20]).astype(np.float32)
    u = (10.0 ** rng.uniform(-5, 38.4, len(g)) * rng.choice([-1, 1], len(g))).astype(np.float32)
    y = gates(act, g, u)
    got, codes_ = gate_of_single_columns(dev, act, g, u)
    seen = np.abs(y) > 1.1e-30
    assert 5000 < seen.sum() < 40000
    assert (np.abs(got - np.abs(y))[seen] <= gate_error(act, g)[seen] * np.abs(y)[seen]).all()
    assert np.array_equal(codes_[seen] >> 7, y[seen] < 0)
    # below 1e-30 the scale is that of 1e-30: half a step of the codes, and y's own error
    below = np.abs(y) < 0.9e-30
    v = y[below] / (1e-30 / 448)
    assert (np.abs(E4M3[codes_[below]] - v) <= np.maximum(2.0 ** -4 * np.abs(v), 2.0 ** -10) + 2.0 ** -19 * np.abs(v) + 1e-12).all()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_a_gate_that_vanishes_leaves_its_block_alone(dev, act, dtype):
    rng = np.random.default_rng(23)
    dim = 256
    g, u = rng.standard_normal((4, dim)), rng.standard_normal((4, dim))
    g[:, ::5] = -100.0 if act == "silu" else -30.0
    u[:, ::5] = 2e38 if dtype == "f32" else 6e4
    g[3] = -110.0 if act == "silu" else -25.0   # a row of nothing else
    x = np.concatenate([g, u], axis=1).astype(np.float32 if dtype == "f32" else np.float16)
    q, s = Out(dev, (4, dim), "u8"), Out(dev, (4, 2), "f32")
    (T.swiglu_rows_fp8 if act == "silu" else T.geglu_rows_fp8)(dev, At(dev, x), q, s, dim, 4)
    y = gates(act, x[:, :dim], x[:, dim:])
    check_codes(q.get(), s.get(), y, 2.0 ** -20 * np.abs(y) + 1e-38)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gates_that_are_no_numbers_mark_their_own_block(dev, act, dtype):
    rng = np.random.default_rng(24)
    dim, rows = 640, 4
    x = rng.standard_normal((rows, 2 * dim))
    bad = np.zeros((rows, 5), bool)
    for r, (b, v) in enumerate(((0, np.inf), (2, -np.inf), (4, np.nan), (1, np.inf))):
        x[r, b * BLOCK + 9 + (r == 3) * dim] = v   # (the last one is an up value)
        bad[r, b] = True
    x = x.astype(np.float32 if dtype == "f32" else np.float16)
    q, s = Out(dev, (rows, dim), "u8"), Out(dev, (rows, 5), "f32")
    (T.swiglu_rows_fp8 if act == "silu" else T.geglu_rows_fp8)(dev, At(dev, x), q, s, dim, rows)
    q, s = q.get(), s.get()
    assert np.array_equal(np.isnan(s), bad) and (q[np.repeat(bad, BLOCK, axis=1)] & 0x7F == 0x7F).all()
    y = np.where(np.repeat(bad, BLOCK, axis=1), 1.0, gates(act, np.nan_to_num(x[:, :dim]), np.nan_to_num(x[:, dim:])))
    for b in range(5):
        good, at = ~bad[:, b], slice(b * BLOCK, (b + 1) * BLOCK)
        check_codes(q[good, at], s[good, b:b + 1], y[good, at], 2.0 ** -18 * np.abs(y[good, at]) + 1e-38)


# (m, n, k, results): ragged everywhere, in each of the tile kernel's forms, with and without ranges of K
NAN_TILES = [(1030, 517, 272, "f16"), (1030, 517, 272, "f32"), (450, 97, 400, "f32"), (450, 130, 1040, "f16"), (333, 3579, 18880, "f16"), (420, 260, 3216, "f32"),
             (1500, 9000, 144, "f16"), (200, 9001, 4112, "f16"), (200, 9001, 4112, "f32")]

NAN_FEW = [(9, 200, 400, "f16"), (16, 517, 8208, "f32"), (30, 260, 656, "f32"), (70, 300, 1168, "f16"), (60, 257, 3216, "f32")]


def test_the_products_with_nans_reach_every_form_of_the_tile_kernel():
    plans = {T.plan_fp8(m, n, k, dtype) for m, n, k, dtype in NAN_TILES}
    assert all(p.startswith("k_fp8_tile") for p in plans), plans
    shapes = {p.split(", ")[0] + p.split(", ")[2] for p in plans}
    assert len(shapes) == 5, shapes
    assert any(p.endswith("splits") for p in plans) and any(p.endswith("1 K-split") for p in plans)
    assert all(T.plan_fp8(m, n, k, dtype).startswith("k_fp8_rows_few") for m, n, k, dtype in NAN_FEW)


@pytest.mark.parametrize("what", ["codes", "row scales", "column scales"])
@pytest.mark.parametrize("m,n,k,dtype", NAN_TILES + NAN_FEW)
def test_nans_stay_in_their_rows_and_columns(dev, m, n, k, dtype, what):
    # a NaN code reaches its row or column, a NaN scale of A its row, one of W its 128 columns, and nothing else; among them the last
    # row and column, in the last block, which K cuts short
    a, a_s, w, w_s = gemm_inputs(np.random.default_rng(m + n + k), m, n, k)
    a_s, w_s = a_s * np.float32(2.0 ** -6), w_s * np.float32(2.0 ** -6)   # (f16 results stay finite)
    want = np.zeros((m, n), bool)
    if what == "codes":
        a[m - 1, k - 1], a[5, 17], w[n - 1, k - 2], w[n // 2, 0] = 0x7F, 0xFF, 0xFF, 0x7F
        want[[m - 1, 5]] = True
        want[:, [n - 1, n // 2]] = True
    elif what == "row scales":
        a_s[m - 1, -1] = a_s[m // 2, 0] = a_s[7, blocks(k) // 2] = np.nan
        want[[m - 1, m // 2, 7]] = True
    else:
        w_s[-1, -1] = w_s[w_s.shape[0] // 2, 0] = np.nan
        for b in (w_s.shape[0] - 1, w_s.shape[0] // 2):
            want[:, b * BLOCK:(b + 1) * BLOCK] = True
    c = Out(dev, (m, n), dtype)
    T.gemm_fp8(dev, At(dev, a), At(dev, a_s), At(dev, w), At(dev, w_s), m, n, k, c)
    got = c.get()
    assert np.array_equal(np.isnan(got), want) and np.isfinite(got[~want]).all()


@pytest.mark.parametrize("m,n,k", [(12, 300, 256), (30, 260, 656), (450, 130, 1040), (1030, 517, 272), (1500, 9000, 144)])
def test_small_products_beside_large_ones_that_cancel(dev, m, n, k):
    # eight features of 448 * 448, -448 * 448 and six ones: f32 results have the six, and rounded by the cast they are f16 results with
    # them; f16 results have them where the plan says f16 instructions, and elsewhere are off by less than 2^-13 of 2^16 a product
    code = {int(v): c for c, v in enumerate(E4M3) if v in (1.0, 448.0, -448.0)}
    a, w = np.full((m, k), code[1], np.uint8), np.full((n, k), code[1], np.uint8)
    a[:, 0::8], a[:, 1::8], w[:, 0::8], w[:, 1::8] = code[448], code[-448], code[448], code[448]
    a_s, w_s = np.ones((m, blocks(k)), np.float32), np.ones((blocks(n), blocks(k)), np.float32)
    inputs = [At(dev, v) for v in (a, a_s, w, w_s)]
    c, half, cast = Out(dev, (m, n), "f32"), Out(dev, (m, n), "f16"), Out(dev, (m, n), "f16")
    T.gemm_fp8(dev, *inputs, m, n, k, c)
    T.gemm_fp8(dev, *inputs, m, n, k, half)
    assert T._lib.load().twm_cast_f32_to_f16(dev.handle, c.ptr, cast.ptr, m * n) == T._lib.OK
    # (whole numbers below 2^24: no sum of them rounds)
    assert (c.get() == k // 8 * 6).all() and (cast.get() == k // 8 * 6).all()
    if "8-bit" in T.plan_fp8(m, n, k, "f16"):
        assert m > 16 and (np.abs(half.get().astype(np.float64) - k // 8 * 6) <= k * 2.0 ** 3).all()
    else:
        assert (half.get() == k // 8 * 6).all()


# ---- the largest sizes that the header allows --------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("m,n", [(1, 40), (16, 5000), (30, 17), (70, 300), (450, 130), (520, 200)])
def test_products_of_the_deepest_rows(dev, m, n, dtype):
    # 2^20 features of ones, the last sixteen 448 in the last row of A and the first of W: sums of whole numbers below 2^24 do not round
    k, code = 1 << 20, {int(v): c for c, v in enumerate(E4M3) if v in (1.0, 448.0)}
    a, w = np.full((m, k), code[1], np.uint8), np.full((n, k), code[1], np.uint8)
    a[-1, -16:], w[0, -16:] = code[448], code[448]
    a_s, w_s = np.full((m, blocks(k)), 2.0 ** -10, np.float32), np.full((blocks(n), blocks(k)), 2.0 ** -10, np.float32)
    c = Out(dev, (m, n), dtype)
    T.gemm_fp8(dev, At(dev, a), At(dev, a_s), At(dev, w), At(dev, w_s), m, n, k, c)
    want = np.ones((m, n))
    want[-1] += 16 * 447 / k
    want[:, 0] += 16 * 447 / k
    want[-1, 0] = 1 + 16 * (448 * 448 - 1) / k
    assert np.array_equal(c.get().astype(np.float64), want.astype(np.float16 if dtype == "f16" else np.float32).astype(np.float64))


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_rows_of_the_most_columns(dev, dtype):
    rows, cols = 2, (1 << 24) - 5
    rng = np.random.default_rng(41)
    x = rng.standard_normal((rows, cols), np.float32).astype(np.float16 if dtype == "f16" else np.float32)
    w = (1 + 0.3 * rng.standard_normal(cols, np.float32)).astype(np.float32)
    q, s, total = Out(dev, (rows, cols), "u8"), Out(dev, (rows, blocks(cols)), "f32"), Out(dev, (rows, cols), "f32")
    T.add_rms_norm_fp8(dev, At(dev, x), None, At(dev, w), 1e-6, rows, cols, q, s, sum=total)
    y = x.astype(np.float64)
    y = y / np.sqrt((y * y).mean(axis=1, keepdims=True) + 1e-6) * w
    q, s = q.get(), s.get()
    assert np.array_equal(total.get(), x.astype(np.float32))
    for at in (slice(0, 1 << 15), slice(8 << 20, (8 << 20) + (1 << 15)), slice((cols >> 7) - 300 << 7, cols)):   # (whole blocks from the first)
        check_codes(q[:, at], s[:, at.start >> 7:blocks(at.stop)], y[:, at], 2.0 ** -20 * np.abs(y[:, at]))
    dim = cols // 2
    x = x.reshape(-1)[:rows * 2 * dim].reshape(rows, 2 * dim)
    q, s = Out(dev, (rows, dim), "u8"), Out(dev, (rows, blocks(dim)), "f32")
    T.swiglu_rows_fp8(dev, At(dev, x), q, s, dim, rows)
    q, s = q.get(), s.get()
    for at in (slice(0, 1 << 15), slice((dim >> 7) - 300 << 7, dim)):
        y = gates("silu", x[:, at], x[:, dim + at.start:dim + at.stop])
        check_codes(q[:, at], s[:, at.start >> 7:blocks(at.stop)], y, 2.0 ** -20 * np.abs(y) + 1e-38)


def test_sample_of_the_most_columns(dev):
    rng = np.random.default_rng(42)
    x = (2 * rng.standard_normal((1, 1 << 24), np.float32)).astype(np.float32)
    x[0, rng.integers(0, 1 << 24, 24)] = 14.0
    for limits in (dict(), dict(p=[0.9]), dict(k=[300], p=[0.95]), dict(k=[100000], mp=[0.001])):
        got, want = draw_tokens(dev, x, rng.random(1), [0.8], **limits)
        assert np.array_equal(got, want), limits
