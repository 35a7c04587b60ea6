"""Attention over a paged key-value cache through the C ABI, against numpy in 64 bits (tolerances: kv_oracle.py)."""
import numpy as np
import pytest

import tensorwarp_amd as T
from kv_oracle import DECODE_STEP, PROMPT_STEP, Pool, attend_rows, check
from test_gpu_fp8 import At, Out

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    with T.WarpDevice(0) as d:
        yield d


def ints(dev, values):
    return T.GpuTensor.from_host(dev, np.asarray(values, np.int32))


def sequences(dev, table, lengths, new=None, first=0):
    starts = None if new is None else ints(dev, first + np.concatenate([[0], np.cumsum(new)]))
    return T.KvSequences(ints(dev, table), ints(dev, lengths), len(lengths), table.shape[1], starts=starts)


def queries(rng, rows, heads, dim):
    return (1.5 * rng.standard_normal((rows, heads, dim))).astype(np.float16)


def run_decode(dev, pool, table, lengths, heads, window=0, scale=None, seed=1, q=None):
    rng, dim = np.random.default_rng(seed), pool.shape[3]
    q = queries(rng, len(lengths), heads, dim) if q is None else q
    out = Out(dev, q.shape, "f16")
    T.attention_decode(dev, pool.upload(dev), sequences(dev, table, lengths), At(dev, q), heads, out, scale=scale, window=window)
    want, tol, _ = attend_rows(pool, table, lengths, [1] * len(lengths), q, dim ** -0.5 if scale is None else scale, window, DECODE_STEP)
    got = out.get()
    check(got, want, tol)
    return got


def run_prompt(dev, pool, table, lengths, new, heads, window=0, scale=None, seed=1, q=None, spare=0, first=0):
    """`first` rows ahead of the sequences' and `spare` behind them belong to none."""
    rng, dim = np.random.default_rng(seed), pool.shape[3]
    rows = sum(new)
    q = queries(rng, rows, heads, dim) if q is None else q
    whole = np.concatenate([queries(rng, first, heads, dim), q, queries(rng, spare, heads, dim)])
    out = Out(dev, whole.shape, "f16")
    T.attention_prompt(dev, pool.upload(dev), sequences(dev, table, lengths, new, first), At(dev, whole), rows + first + spare, heads, out, scale=scale,
                       window=window)
    want, tol, _ = attend_rows(pool, table, lengths, new, q, dim ** -0.5 if scale is None else scale, window, PROMPT_STEP)
    got = out.get()
    untouched = np.concatenate([got[:first], got[first + rows:]]).view(np.uint16)
    assert (untouched == 12345).all()
    check(got[first:first + rows], want, tol)
    return got[first:first + rows]


HEADS = [(1, 1), (14, 2), (28, 4), (6, 6), (40, 2), (5, 1)]
LENGTHS = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 255, 257, 300, 511, 640, 1000]


@pytest.mark.parametrize("cache", ["f16", "e4m3"])
@pytest.mark.parametrize("dim,page", [(64, 16), (128, 16), (128, 64), (256, 32), (64, 256), (128, 128)])
@pytest.mark.parametrize("heads,kv", HEADS)
def test_decode(dev, heads, kv, dim, page, cache):
    pool = Pool(np.random.default_rng(heads + dim + page), 4200 // page + 2 * len(LENGTHS), kv, page, dim, cache)
    run_decode(dev, pool, pool.fill(LENGTHS), LENGTHS, heads)


@pytest.mark.parametrize("cache", ["f16", "e4m3"])
@pytest.mark.parametrize("window", [1, 7, 64, 100, 500])
def test_decode_looks_back_a_window(dev, window, cache):
    pool = Pool(np.random.default_rng(window), 600, 2, 16, 128, cache, scales=window != 7)
    table = pool.fill(LENGTHS)
    for s, n in enumerate(LENGTHS):   # pages behind the window are gone
        table[s, :max(0, n - window) // 16] = -1
    run_decode(dev, pool, table, LENGTHS, 14, window=window)


@pytest.mark.parametrize("cache", ["f16", "e4m3"])
@pytest.mark.parametrize("seqs,longest", [(1, 20000), (3, 9001), (70, 300)])
def test_decode_of_few_and_of_many_sequences(dev, seqs, longest, cache):
    rng = np.random.default_rng(seqs)
    lengths = [longest] + list(rng.integers(0, longest, seqs - 1))
    pool = Pool(rng, sum(-(-n // 64) for n in lengths), 2, 64, 64, cache)
    a = run_decode(dev, pool, pool.fill(lengths), lengths, 14)
    assert a.shape[0] == seqs


def test_decode_is_deterministic(dev):
    rng = np.random.default_rng(3)
    lengths = [4000, 100, 2500]
    pool = Pool(rng, 500, 4, 16, 128)
    table = pool.fill(lengths)
    first = run_decode(dev, pool, table, lengths, 28)
    for _ in range(3):
        assert np.array_equal(run_decode(dev, pool, table, lengths, 28).view(np.uint16), first.view(np.uint16))


PROMPTS = [  # (new, tokens in the cache with them)
    ([1], [1]), ([5], [5]), ([37], [37]), ([64], [64]), ([65, 1, 0, 130], [65, 1, 0, 130]), ([200, 3], [200, 700]), ([16, 16, 16], [300, 16, 33]),
    ([1, 1, 1, 1], [1, 64, 65, 500]), ([4, 9, 2], [129, 128, 127]), ([0, 0, 7], [0, 5, 7]), ([300], [999])]


@pytest.mark.parametrize("cache", ["f16", "e4m3"])
@pytest.mark.parametrize("dim,page,heads,kv", [(64, 16, 14, 2), (128, 16, 28, 4), (128, 64, 3, 3), (256, 32, 4, 2), (128, 256, 20, 1), (64, 128, 5, 5)])
@pytest.mark.parametrize("new,lengths", PROMPTS)
def test_prompt(dev, new, lengths, dim, page, heads, kv, cache):
    pool = Pool(np.random.default_rng(sum(new) + dim), sum(-(-n // page) for n in lengths) + 3, kv, page, dim, cache)
    run_prompt(dev, pool, pool.fill(lengths), lengths, new, heads)


@pytest.mark.parametrize("cache", ["f16", "e4m3"])
@pytest.mark.parametrize("window", [1, 5, 64, 65, 200])
def test_prompt_looks_back_a_window(dev, window, cache):
    new, lengths = [150, 20, 1, 90], [400, 20, 300, 90]
    pool = Pool(np.random.default_rng(window), 80, 2, 16, 128, cache)
    table = pool.fill(lengths)
    for s, (n, length) in enumerate(zip(new, lengths)):
        table[s, :max(0, length - n + 1 - window) // 16] = -1
    run_prompt(dev, pool, table, lengths, new, 8, window=window)


@pytest.mark.parametrize("cache", ["f16", "e4m3"])
@pytest.mark.parametrize("dim,heads,kv,window", [(64, 14, 2, 0), (128, 7, 1, 0), (128, 4, 4, 2500), (256, 4, 2, 0)])
@pytest.mark.parametrize("new,lengths", [([1], [6000]), ([5], [4003]), ([40, 2, 1], [3000, 90, 5001]), ([150], [4500])])
def test_few_rows_behind_many_tokens(dev, new, lengths, dim, heads, kv, window, cache):
    # shared out among workgroups by their tokens, in as many parts as a sequence has tiles for
    pool = Pool(np.random.default_rng(sum(new) + dim), sum(-(-n // 64) for n in lengths) + 3, kv, 64, dim, cache)
    table = pool.fill(lengths)
    table[0, 20:25] = -1   # (absent pages, and rows whose parts lack them all or see none of theirs)
    run_prompt(dev, pool, table, lengths, new, heads, window=window)


def test_rows_of_no_sequence_stay_as_they_were(dev):
    pool = Pool(np.random.default_rng(8), 40, 2, 16, 64)
    run_prompt(dev, pool, pool.fill([40, 3, 70]), [40, 3, 70], [33, 0, 70], 6, first=5, spare=150)


def test_rows_without_tokens_are_zeros(dev):
    # more rows than tokens: the first ones precede the sequence
    pool = Pool(np.random.default_rng(9), 40, 2, 16, 128)
    got = run_prompt(dev, pool, pool.fill([3, 0, 70]), [3, 0, 70], [10, 4, 75], 4)
    assert (got[:7] == 0).all() and (got[10:14] == 0).all() and (got[14:19] == 0).all()
    got = run_decode(dev, pool, np.full((3, 2), -1, np.int32), [20, -5, 0], 4)
    assert (got == 0).all()


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("cache", ["f16", "e4m3"])
def test_absent_pages_take_no_part(dev, cache, dim):
    lengths = [200, 90, 64, 700]
    pool = Pool(np.random.default_rng(10), 80, 2, 16, dim, cache)
    table = pool.fill(lengths)
    table[0, 3], table[0, 12], table[1, 0], table[2, :] = -1, 80, 1 << 30, -7
    table[3, 5:20] = -(1 << 31)
    run_decode(dev, pool, table, lengths, 6)
    run_prompt(dev, pool, table, lengths, [150, 90, 5, 400], 6)
    # a table that is too short for its sequences
    run_decode(dev, pool, np.ascontiguousarray(table[:, :4]), lengths, 6)
    run_prompt(dev, pool, np.ascontiguousarray(table[:, :4]), lengths, [150, 90, 5, 30], 6)


@pytest.mark.parametrize("width", [None, 40])
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_what_a_row_does_not_see_does_not_reach_it(dev, dim, bad, width):
    # later tokens of the same prompt, earlier ones behind the window, other sequences' pages: infinities and NaN in all of them
    new = lengths = [150, 40]
    pool = Pool(np.random.default_rng(11), 30, 2, 16, dim)
    table = pool.fill(lengths, width)
    for name, tokens in (("v", (70, 149)), ("k", (90,)), ("v", (10,))):
        for t in tokens:
            pool.bits[name][table[0, t // 16], 1, t % 16, 5::17] = np.float16(bad).view(np.uint16)
    got = run_prompt(dev, pool, table, lengths, new, 4, window=30)
    assert np.isfinite(got[:10].astype(np.float64)).all() and np.isfinite(got[150:].astype(np.float64)).all()
    assert not np.isfinite(got[149].astype(np.float64)).all()
    got = run_decode(dev, pool, table, [70, 40], 4, window=30)   # (token 70 is the first that is not there)
    assert np.isfinite(got.astype(np.float64)).all()


@pytest.mark.parametrize("width", [None, 40])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_infinite_scores_and_values_are_as_the_formula_has_them(dev, dim, width):
    pool = Pool(np.random.default_rng(12), 30, 1, 16, dim)
    lengths = [100, 100, 100]
    table = pool.fill(lengths, width)
    pool.bits["v"][table[0, 2], 0, 3, 7] = np.float16(np.inf).view(np.uint16)    # one value: that column is infinite
    pool.bits["v"][table[1, 2], 0, 3, 7] = np.float16(np.nan).view(np.uint16)
    pool.bits["k"][table[2, 2], 0, 3, 7] = np.float16(np.nan).view(np.uint16)    # a score: the whole row is NaN
    got = run_decode(dev, pool, table, lengths, 2)
    assert np.isposinf(got[0, :, 7]).all() and np.isnan(got[1, :, 7]).all() and np.isnan(got[2]).all() and np.isfinite(got[0, :, 8]).all()
    run_prompt(dev, pool, table, lengths, [100, 100, 100], 2)


@pytest.mark.parametrize("width", [None, 40])
@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("scale", [1e-3, 1.0, 30.0])
def test_scales_and_large_scores(dev, scale, dim, width):
    # scores of thousands: one token takes all the weight; far apart from one another in the order that raises the maximum most often
    pool = Pool(np.random.default_rng(13), 60, 2, 16, dim)
    lengths = [400, 33, 200]
    table = pool.fill(lengths, width, spread=4.0)
    run_decode(dev, pool, table, lengths, 4, scale=scale)
    run_prompt(dev, pool, table, lengths, [300, 33, 1], 4, scale=scale)


@pytest.mark.parametrize("width", [None, 40])
@pytest.mark.parametrize("dim", [128, 256])
def test_rising_scores(dev, dim, width):
    # every token outweighs the ones before it, by up to 2^20
    n = 500
    pool = Pool(np.random.default_rng(14), 40, 1, 16, dim)
    table = pool.fill([n], width)
    q = np.ones((n, 1, dim), np.float16)
    for t in range(n):
        pool.bits["k"][table[0, t // 16], 0, t % 16] = np.float16(t * 0.11).view(np.uint16)
    run_decode(dev, pool, table, [n], 1, scale=1.0, q=q[:1])
    run_prompt(dev, pool, table, [n], [n], 1, scale=1.0, q=q)


@pytest.mark.parametrize("skip,q_more,out_more", [(1, 3, 0), (3, 0, 5), (5, 8, 16)])
def test_strides_and_odd_addresses(dev, skip, q_more, out_more):
    rng, heads, dim = np.random.default_rng(15), 6, 64
    lengths, new = [70, 33, 5], [20, 33, 2]
    pool = Pool(rng, 20, 2, 16, dim)
    table, width = pool.fill(lengths), heads * dim
    rows = sum(new)
    q = queries(rng, rows, heads, dim)
    wide = np.full((rows, width + q_more), np.nan, np.float16)
    wide[:, :width] = q.reshape(rows, width)
    for call, per_seq, step in ((T.attention_prompt, new, PROMPT_STEP), (T.attention_decode, [1, 1, 1], DECODE_STEP)):
        n = sum(per_seq)
        out = Out(dev, (n, width + out_more), "f16")
        more = [] if call is T.attention_decode else [n]
        call(dev, pool.upload(dev), sequences(dev, table, lengths, per_seq), At(dev, wide[:n], skip), *more, heads, out, q_stride=width + q_more if q_more else 0,
             out_stride=width + out_more if out_more else 0)
        want, tol, _ = attend_rows(pool, table, lengths, per_seq, q[:n], dim ** -0.5, 0, step)
        got = out.get()
        assert (got[:, width:].view(np.uint16) == 12345).all()
        check(got[:, :width].reshape(want.shape), want, tol)


def test_nothing_to_do(dev):
    pool = Pool(np.random.default_rng(16), 4, 1, 16, 64)
    cache, empty = pool.upload(dev), T.GpuTensor.from_host(dev, np.zeros(64, np.int32))
    out = Out(dev, (2, 64), "f16")
    T.attention_decode(dev, cache, T.KvSequences(empty, empty, 0, 0), At(dev, np.zeros((1, 64), np.float16)), 1, out)
    T.attention_prompt(dev, cache, T.KvSequences(empty, empty, 0, 0, starts=empty), At(dev, np.zeros((1, 64), np.float16)), 2, 1, out)
    assert (out.get().view(np.uint16) == 12345).all()
    T.attention_decode(dev, cache, T.KvSequences(empty, ints(dev, [5, 9]), 2, 0), At(dev, np.ones((2, 64), np.float16)), 1, out)   # tables of no pages
    assert (out.get() == 0).all()
