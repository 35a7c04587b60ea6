"""Attention over a paged key-value cache whose scores are large, up to the largest that finite f16 queries and keys make.  What a row comes to is
known there whatever a score's own roundings are: one token's value where it sees one, or where one outweighs all others by far; the mean where
all scores are the same sum of the same products; the formula on differences where every partial sum of the scores is exact."""
import numpy as np
import pytest

import tensorwarp_amd as T
from kv_oracle import DECODE_STEP, PROMPT_STEP, Pool, half_step_f16
from test_gpu_attention import sequences
from test_gpu_fp8 import At, Out

pytestmark = pytest.mark.gpu

# a short table and a wide one: a workgroup for each sequence or shares of all, waves in pairs or not (heads of 256 values are always in pairs)
WIDTHS = [None, 400]
TINY = 2.0 ** -20   # roundings in 32 bits: of the scale of values, of the weights' exponential, of the division by their sum


@pytest.fixture(scope="module")
def dev():
    with T.WarpDevice(0) as d:
        yield d


def run(dev, kc, seqs, q, heads, **more):
    out = Out(dev, q.shape, "f16")
    if seqs.starts is None:
        T.attention_decode(dev, kc, seqs, At(dev, q), heads, out, **more)
    else:
        T.attention_prompt(dev, kc, seqs, At(dev, q), q.shape[0], heads, out, **more)
    return out.get().astype(np.float64)


def near(got, want, tol):
    assert np.isfinite(got).all()
    off = np.abs(got - want) / (tol + half_step_f16(want))
    assert off.max() <= 1.0, (off.max(), (off > 1).sum(), off.size)


def filled(seed, dim, cache, n, width, keys):
    """One sequence of n tokens whose values are random and whose keys (f16) `keys` gives, of one key-value head with pages of 16."""
    pool = Pool(np.random.default_rng(seed), -(-n // 16) + 2, 1, 16, dim, cache, scales=False)
    table = pool.fill([n], width)
    if cache == "f16":
        for t in range(n):
            pool.bits["k"][table[0, t // 16], 0, t % 16] = keys[t].astype(np.float16).view(np.uint16)
    return pool, table


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("cache", ["f16", "e4m3"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("size", [700.0, 2000.0, 3001.0, 4000.0, 10007.0, 40000.0, 65504.0])
@pytest.mark.parametrize("sign", [1, -1])
def test_a_row_that_sees_one_token_is_its_value(dev, size, sign, dim, cache, width):
    # every row of 70 looks back one token.  e4m3 keys are as large as they come with the scales that make them so
    n, heads = 70, 2
    rng = np.random.default_rng(int(size) + dim)
    pool, table = filled(int(size) + dim, dim, cache, n, width, np.full((n, dim), size))
    if cache == "e4m3":
        pool.bits["k"][:, 0] = np.where(rng.random((pool.shape[0], 16, dim)) < 0.5, 0x7E, 0x7D)   # 448 and 416
        pool.scales = {"k": np.full(1, size / 448.0, np.float32), "v": np.full(1, 0.0371, np.float32)}
    q = (sign * size * rng.choice([1.0, 1.0, 0.75], (n, heads, dim))).astype(np.float16)
    v = np.repeat(pool.tokens("v", table[0], n).transpose(1, 0, 2), heads, axis=1)
    kc = pool.upload(dev)
    near(run(dev, kc, sequences(dev, table, [n], [n]), q, heads, window=1), v, TINY * np.abs(v))
    each = np.arange(1, n + 1)
    near(run(dev, kc, sequences(dev, np.repeat(table, n, axis=0), each), q, heads, window=1), v, TINY * np.abs(v))


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("size", [700.0, 2000.0, -3001.0, 10007.0, -40000.0, 65504.0])
def test_equal_scores_are_the_mean(dev, size, dim, width):
    # (the same products in the same order: scores are equal to the bit whatever their roundings are)
    n, heads = 200, 3
    pool, table = filled(3, dim, "f16", n, width, np.full((n, dim), abs(size)))
    q = np.full((n, heads, dim), size, np.float16)
    v = pool.tokens("v", table[0], n)[0]
    counts = np.arange(1, n + 1)[:, None]
    mean, magnitude = v.cumsum(0) / counts, np.abs(v).cumsum(0) / counts
    for rows, seqs in ((slice(None), sequences(dev, table, [n], [n])), (slice(n - 1, n), sequences(dev, table, [n]))):
        got = run(dev, pool.upload(dev), seqs, q[rows], heads)
        near(got, np.repeat(mean[rows, None], heads, 1), np.repeat((((n + 16) * 2.0 ** -23 + TINY) * magnitude)[rows, None], heads, 1))


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("size", [200.0, 2000.0, 4000.0, 40000.0])
@pytest.mark.parametrize("at", [0, 63, 64, 130, 399])
def test_one_token_that_outweighs_all_others(dev, at, size, dim, width):
    # others score 0, or a tenth of it; the one comes first, later in the first tile, in later ones and last
    n, heads = 400, 2
    rng = np.random.default_rng(at)
    keys = np.where(rng.random((n, 1)) < 0.5, 0.0, size / 10) * np.ones((n, dim))
    keys[at] = size
    pool, table = filled(at, dim, "f16", n, width, keys)
    q = np.full((n - at, heads, dim), size, np.float16)
    v = pool.tokens("v", table[0], n)[0, at]
    for rows, seqs in ((n - at, sequences(dev, table, [n], [n - at])), (1, sequences(dev, table, [n]))):
        got = run(dev, pool.upload(dev), seqs, q[:rows], heads)
        near(got, np.broadcast_to(v, got.shape), TINY * np.abs(v))


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("offset", [0, 1 << 10, 1 << 12, 1 << 13, 1 << 16, 1 << 19, 1 << 22, 1 << 25, -(1 << 16), -(1 << 25)])
def test_differences_beside_a_large_sum_of_products(dev, offset, dim, width):
    # scores offset + gap, gaps whole multiples of 4 from -60 to 60: every sum is exact in 32 bits.  Scaled, they are up to 15 apart and come in an
    # order that raises the maximum now and then
    n, heads, group = 333, 2, 16
    rng = np.random.default_rng(abs(offset) % 1000 + dim)
    gaps = 4.0 * rng.integers(0, group, n) - 60.0 * (np.arange(n) < 250) * (rng.random(n) < 0.9)
    keys = np.zeros((n, dim))
    keys[:, 0], keys[:, dim - 3] = abs(offset) / 4096.0 if offset else 0.0, gaps
    pool, table = filled(dim, dim, "f16", n, width, keys)
    q = np.zeros((n, heads, dim), np.float16)
    q[:, :, 0], q[:, :, dim - 3] = np.sign(offset) * 4096.0, 1.0
    v = pool.tokens("v", table[0], n)[0]
    p = np.exp(0.125 * (gaps - gaps.max()))
    total = p.cumsum()[:, None]
    want, magnitude = (p[:, None] * v).cumsum(0) / total, (p[:, None] * np.abs(v)).cumsum(0) / total
    # an exponent of up to 21.7 in base 2: half a step (2^-20) of its own, 2^-23 of it from the scale's roundings, as much again where the maximum was raised,
    # together below 2^-17; twice over, for the weight and the sum, and the exponential's own: 2^-16.  In f16 2^-25 at least, of a weight 2^8
    for rows, seqs, step in ((slice(None), sequences(dev, table, [n], [n]), PROMPT_STEP), (slice(n - 1, n), sequences(dev, table, [n]), DECODE_STEP)):
        got = run(dev, pool.upload(dev), seqs, q[rows], heads, scale=0.125)
        tol = ((step + 2.0 ** -16 + (n + 16) * 2.0 ** -23) * magnitude + 2.0 ** -33 * np.abs(v).sum(0))[rows]
        near(got, np.repeat(want[rows, None], heads, 1), np.repeat(tol[:, None], heads, 1))


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("cache", ["f16", "e4m3"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("scale,k_scale", [(3.0e38, 1.0), (3.4e38, 0.03), (1.0e-38, 1.0), (1.5e-45, 1.0), (1.0, 3.0e38), (1.0e-30, 1.0e-30)])
def test_the_largest_and_the_smallest_scales(dev, scale, k_scale, dim, cache, width):
    # whole scores, so that differences are at least 1 or none: of the largest scales only the largest scores count, alike, of the smallest all do
    n, heads = 150, 2
    rng = np.random.default_rng(dim)
    scores = rng.integers(-8, 4, n)
    keys = np.zeros((n, dim))
    keys[:, dim - 5] = scores
    pool, table = filled(dim, dim, cache, n, width, keys)
    if cache == "e4m3":
        pool.scales["k"] = np.full(1, k_scale, np.float32)
        codes = {0: 0, 1: 0x38, 2: 0x40, 3: 0x44, 4: 0x48, 5: 0x4A, 6: 0x4C, 7: 0x4E, 8: 0x50}   # e4m3 of the whole numbers up to 8
        for t in range(n):
            pool.bits["k"][table[0, t // 16], 0, t % 16] = 0
            pool.bits["k"][table[0, t // 16], 0, t % 16, dim - 5] = codes[abs(scores[t])] | (0x80 if scores[t] < 0 else 0)
    elif k_scale != 1.0:
        return
    q = np.zeros((n, heads, dim), np.float16)
    q[:, :, dim - 5] = 1.0
    v = pool.tokens("v", table[0], n)[0]
    want, magnitude = np.zeros((n, dim)), np.zeros((n, dim))
    for row in range(n):
        seen = scores[:row + 1]
        of = v[:row + 1][seen == seen.max()] if scale * k_scale > 1.0 else v[:row + 1]
        want[row], magnitude[row] = of.mean(0), np.abs(of).mean(0)
    for rows, seqs in ((slice(None), sequences(dev, table, [n], [n])), (slice(n - 1, n), sequences(dev, table, [n]))):
        got = run(dev, pool.upload(dev), seqs, q[rows], heads, scale=scale)
        near(got, np.repeat(want[rows, None], heads, 1), np.repeat((((n + 16) * 2.0 ** -23 + TINY) * magnitude)[rows, None], heads, 1))


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("up", [100, -100])
def test_a_scale_of_scores_and_one_of_keys_that_meet_in_the_middle(dev, up, dim, width):
    # 2^up times 2^-up of both: the same bits as without
    n, heads = 90, 4
    pool, table = filled(1, dim, "e4m3", n, width, None)
    q = (1.5 * np.random.default_rng(2).standard_normal((n, heads, dim))).astype(np.float16)
    results = []
    for scale, k_scale in ((0.125, 0.03125), (0.125 * 2.0 ** up, 0.03125 * 2.0 ** -up)):
        pool.scales["k"] = np.full(1, k_scale, np.float32)
        kc = pool.upload(dev)
        results.append([run(dev, kc, s, rows, heads, scale=scale) for s, rows in ((sequences(dev, table, [n], [n]), q), (sequences(dev, table, [n]), q[:1]))])
    for a, b in zip(*results):
        assert np.isfinite(a).all() and np.array_equal(a, b)


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("value", [3.0, 60000.0])
@pytest.mark.parametrize("infinite", [False, True])
def test_tokens_without_weight_add_nothing(dev, infinite, value, dim, width):
    # one token, the second, outweighs a thousand others by e^200: 0 in 32 bits.  Its value is the result, zeros in all but one column, however large the others' are.
    # With an infinite one among them, in a column of its own and with a weight of its own, rows that do not see it stay as they are
    n, heads = 1000, 2
    pool = Pool(np.random.default_rng(1), 70, 1, 16, dim)
    table = pool.fill([n], width)
    bits = lambda x: np.float16(x).view(np.uint16)
    at = lambda t: (table[0, t // 16], 0, t % 16)
    for t in range(n):
        pool.bits["k"][at(t)], pool.bits["v"][at(t)] = 0, bits(value)
    pool.bits["k"][at(1)][7], pool.bits["v"][at(1)] = bits(200.0), 0
    pool.bits["v"][at(1)][9] = bits(0.375)
    if infinite:
        pool.bits["k"][at(600)][7], pool.bits["v"][at(600)][11] = bits(198.0), bits(np.inf)
        pool.bits["v"][at(600)][12] = 0
    q = np.zeros((n - 1, heads, dim), np.float16)
    q[:, :, 7] = 1.0
    want = np.zeros(dim)
    want[9] = 0.375
    for rows, seqs in ((n - 1, sequences(dev, table, [n], [n - 1])), (1, sequences(dev, table, [n]))):
        got = run(dev, pool.upload(dev), seqs, q[:rows], heads, scale=1.0)
        if not infinite:
            assert np.array_equal(got, np.broadcast_to(want, got.shape))
            continue
        # rows from the infinite token on: its column is infinite; column 12, which it and the first have zeros in, has 2^-38 of the others' at most
        behind = slice(599, None) if rows > 1 else slice(None)
        assert np.isposinf(got[behind, :, 11]).all()
        assert np.abs(got[behind, :, 12]).max() <= n * 2.0 ** -38 * value + 2.0 ** -25
        if rows > 1:
            assert np.array_equal(got[:599], np.broadcast_to(want, got[:599].shape))


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("cache", ["f16", "e4m3"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("scale", [1.0, 30.0, 1000.0])
def test_random_scores_of_thousands_and_more(dev, scale, dim, cache, width):
    # Results are means of values that are seen, whatever the weights; and where one score leads by more than all roundings of both (dim steps of 2^-23 of
    # sum |q k|, each) and 30 besides, the others together weigh less than n e^-30 and the result is its value
    n, heads, kv = 300, 4, 2
    pool = Pool(np.random.default_rng(dim), 24, kv, 16, dim, cache)
    table = pool.fill([n], width, spread=4.0)
    q = (1.5 * np.random.default_rng(int(scale)).standard_normal((n, heads, dim))).astype(np.float16)
    k, v = (np.repeat(pool.tokens(name, table[0], n), heads // kv, axis=0) for name in "kv")
    for first, seqs in ((0, sequences(dev, table, [n], [n])), (n - 1, sequences(dev, table, [n]))):
        got = run(dev, pool.upload(dev), seqs, q[first:], heads, scale=scale)
        leading = 0
        for i, row in enumerate(range(first, n)):
            seen = v[:, :row + 1]
            low, high = seen.min(1), seen.max(1)
            room = TINY * np.abs(seen).max(1)
            assert (got[i] >= low - room - half_step_f16(low)).all() and (got[i] <= high + room + half_step_f16(high)).all(), row
            products = k[:, :row + 1] * q[row][:, None].astype(np.float64)
            s, off = scale * products.sum(2), scale * dim * 2.0 ** -23 * np.abs(products).sum(2).max(1)
            for h in range(heads):
                order = np.argsort(s[h])
                if row == 0 or s[h, order[-1]] - s[h, order[-2]] > 2 * off[h] + 30.0:
                    leading += 1
                    near(got[i, h], seen[h, order[-1]], room[h] + (row + 1) * np.exp(-30.0) * 2 * np.abs(seen[h]).max(0))
        assert leading > 0.75 * len(got) * heads or first or scale < 30.0   # (counted on the host: 982 to 1200 of 1200)


@pytest.mark.parametrize("cache", ["f16", "e4m3"])
@pytest.mark.parametrize("dim,heads", [(64, 1), (128, 1), (128, 8), (256, 2)])
@pytest.mark.parametrize("every", [1, 32, 40, 100])
def test_rows_of_large_and_of_small_scores_in_turn(dev, every, dim, heads, cache):
    # rows whose scores have 2^20 added, and rows without, in turn by `every` rows times heads: some waves of a workgroup have such rows and others do not.
    # What a row comes to is the same; longer than a tile's buffers live, and each token has a value of its own
    n = 900
    rng = np.random.default_rng(every + dim)
    gaps = 4.0 * rng.integers(0, 16, n)
    pool, table = filled(dim, dim, cache, n, 80, np.zeros((n, dim)))
    large = 8192.0 if cache == "f16" else 448.0
    for t in range(n):
        at = table[0, t // 16], 0, t % 16
        pool.bits["k"][at] = 0
        if cache == "f16":
            pool.bits["k"][at][[0, dim - 3]] = np.array([large, gaps[t]], np.float16).view(np.uint16)
        else:   # e4m3: 448 and 0, 8, ... 56 (of three bits), so that sums are exact as well
            gaps[t] = 8.0 * (gaps[t] // 8)
            codes = {0: 0x00, 8: 0x50, 16: 0x58, 24: 0x5C, 32: 0x60, 40: 0x62, 48: 0x64, 56: 0x66}
            pool.bits["k"][at][[0, dim - 3]] = 0x7E, codes[int(gaps[t])]
    q = np.zeros((n, heads, dim), np.float16)
    q[:, :, dim - 3] = 1.0
    added = (np.arange(n * heads).reshape(n, heads) // every) % 2 == 1
    q[added, 0] = 128.0 if cache == "f16" else 2048.0
    v = pool.tokens("v", table[0], n)[0]
    p = np.exp(0.125 * (gaps - gaps.max()))
    total = p.cumsum()[:, None]
    want, magnitude = (p[:, None] * v).cumsum(0) / total, (p[:, None] * np.abs(v)).cumsum(0) / total
    # (as above, and rows without the addition have exponents rounded at up to 2^10: 2^-15, where the maximum was raised too, for the weight and the sum)
    tol = (PROMPT_STEP + 2.0 ** -12 + (n + 16) * 2.0 ** -23) * magnitude + 2.0 ** -33 * np.abs(v).sum(0)
    kc = pool.upload(dev)
    for _ in range(3):
        got = run(dev, kc, sequences(dev, table, [n], [n]), q, heads, scale=0.125)
        near(got, np.repeat(want[:, None], heads, 1), np.repeat(tol[:, None], heads, 1))
