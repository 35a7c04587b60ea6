"""Attention over a paged key-value cache where its kernels change their way of sharing the work, and at the ends of its ranges: short
and long tables, many sequences, groups of more heads than a matrix instruction has columns, windows of any size, hundreds of thousands
of tokens, pools beyond 32-bit offsets, calls of thousands of rows, two contexts at once."""
import numpy as np
import pytest

import tensorwarp_amd as T
from kv_oracle import DECODE_STEP, PROMPT_STEP, Pool, attend_rows, check, half_step_f16
from test_gpu_attention import queries, run_decode, run_prompt, sequences
from test_gpu_fp8 import At, Out

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    with T.WarpDevice(0) as d:
        yield d


def widened(table, width):
    return np.ascontiguousarray(np.pad(table, ((0, 0), (0, width - table.shape[1])), constant_values=-1))


# (short tables: a workgroup has a sequence to itself; wide ones, whatever the lengths: shares and a join)
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("cache", ["f16", "e4m3"])
@pytest.mark.parametrize("heads,kv,dim,page", [(1, 1, 64, 16), (17, 1, 64, 32), (33, 1, 128, 16), (14, 2, 128, 64), (12, 3, 256, 16), (32, 32, 64, 16), (130, 2, 64, 16)])
def test_decode_with_short_and_wide_tables(dev, heads, kv, dim, page, cache, wide):
    lengths = [0, 1, 31, 32, 33, 64, 100, 129, -3, 200, 255, 256]
    pool = Pool(np.random.default_rng(heads + dim), 1200 // page + 14, kv, page, dim, cache)
    table = pool.fill(lengths)
    run_decode(dev, pool, widened(table, 20000 // page) if wide else table, lengths, heads)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("cache", ["f16", "e4m3"])
@pytest.mark.parametrize("window", [1, 33, 400])
def test_decode_windows_over_long_tables(dev, window, cache, dim):
    # what a window leaves decides the sharing, not the table; windows that begin inside a page and a step
    lengths = [4000, 1, 33, 2047, 2048, 399, 401]
    pool = Pool(np.random.default_rng(window + dim), 600, 2, 16, dim, cache)
    run_decode(dev, pool, pool.fill(lengths), lengths, 6, window=window)


@pytest.mark.parametrize("window", [0x7FFFFFFF, 0x80000000, 0xFFFFFFFF])
def test_windows_larger_than_any_sequence(dev, window):
    lengths = [300, 5, 0, -7]
    pool = Pool(np.random.default_rng(1), 40, 2, 16, 64)
    table = pool.fill(lengths)
    run_decode(dev, pool, table, lengths, 4, window=window)
    run_prompt(dev, pool, table, lengths, [100, 5, 0, 0], 4, window=window)


@pytest.mark.parametrize("seqs,longest,wide", [(64, 40, False), (65, 40, True), (300, 20, False), (300, 20, True), (1500, 3, False), (1500, 3, True), (129, 700, True)])
def test_decode_of_many_sequences(dev, seqs, longest, wide):
    rng = np.random.default_rng(seqs)
    lengths = list(rng.integers(0, longest + 1, seqs))
    pool = Pool(rng, sum(-(-n // 16) for n in lengths) + 1, 2, 16, 64)
    table = pool.fill(lengths)
    run_decode(dev, pool, widened(table, 500) if wide else table, lengths, 4)


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("seqs,most,behind", [(64, 4, 30), (4097, 1, 3), (65, 4, 30), (300, 3, 100), (1100, 2, 5), (130, 40, 0)])
def test_prompts_of_many_sequences(dev, seqs, most, behind, dim, wide):
    rng = np.random.default_rng(seqs)
    new = list(rng.integers(0, most + 1, seqs))
    lengths = [n + int(rng.integers(0, behind + 1)) for n in new]
    pool = Pool(rng, sum(-(-n // 16) for n in lengths) + 1, 1, 16, dim)
    table = pool.fill(lengths)
    run_prompt(dev, pool, widened(table, 40) if wide else table, lengths, new, 3, first=2, spare=9)


# (tables of 512 tokens and wider ones: waves in pairs, and not)
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("cache", ["f16", "e4m3"])
@pytest.mark.parametrize("dim,heads,kv,page", [(64, 6, 2, 16), (128, 7, 1, 64), (128, 4, 4, 16)])
@pytest.mark.parametrize("window", [0, 50])
def test_prompts_with_short_and_wide_tables(dev, dim, heads, kv, page, cache, window, wide):
    new, lengths = [3, 0, 70, 1, 130, 64], [3, 5, 200, 450, 130, 512]
    pool = Pool(np.random.default_rng(dim + heads), 1400 // page + 8, kv, page, dim, cache)
    table = pool.fill(lengths)
    table[2, 1] = -1
    run_prompt(dev, pool, widened(table, 2000 // page) if wide else table, lengths, new, heads, window=window, first=1, spare=4)


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("heads,kv", [(17, 1), (130, 1), (66, 2)])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_prompt_with_heads_across_the_rows_of_a_workgroup(dev, heads, kv, dim, wide):
    new, lengths = [5, 30, 1], [5, 90, 70]
    pool = Pool(np.random.default_rng(heads), 16, kv, 16, dim)
    table = pool.fill(lengths)
    run_prompt(dev, pool, widened(table, 50) if wide else table, lengths, new, heads)


@pytest.mark.parametrize("cache", ["f16", "e4m3"])
def test_hundreds_of_thousands_of_tokens(dev, cache):
    lengths = [250001, 3]
    pool = Pool(np.random.default_rng(2), 250001 // 256 + 3, 1, 256, 64, cache)
    table = pool.fill(lengths)
    run_decode(dev, pool, table, lengths, 3)
    run_prompt(dev, pool, table, lengths, [2, 1], 3)


@pytest.mark.parametrize("cache", ["f16", "e4m3"])
def test_hundreds_of_millions_of_tokens(dev, cache):
    # one page of 256 tokens named a million times is that page's attention.  Every token is one of 2^28 and no more than (2^28 / 2048 waves + 64)
    # f32 additions stand behind a sum, of products and of weights
    pool = Pool(np.random.default_rng(9), 3, 1, 256, 64, cache)
    table = np.full((2, 1 << 20), pool.fill([256])[0, 0], np.int32)
    lengths, heads = [1 << 28, 256], 2
    q = queries(np.random.default_rng(10), 2, heads, 64)
    kc, seqs = pool.upload(dev), sequences(dev, table, lengths, [1, 1])
    for call, more in ((T.attention_decode, []), (T.attention_prompt, [2])):
        out = Out(dev, q.shape, "f16")
        call(dev, kc, seqs, At(dev, q), *more, heads, out)
        want, tol, _ = attend_rows(pool, table[:, :1], [256, 256], [1, 1], q, 0.125, 0, PROMPT_STEP)
        most = np.abs(pool.tokens("v", table[0, :1], 256)).max(1)[None]
        tol[0] += 2 * (131072 + 64) * 2.0 ** -23 * most[0]
        check(out.get(), want, tol)


@pytest.mark.parametrize("dim,heads,kv,cache", [(64, 2, 1, "f16"), (128, 2, 2, "e4m3"), (256, 2, 1, "f16")])
@pytest.mark.parametrize("window", [0, 777])
def test_thousands_of_rows_against_their_single_tokens(dev, dim, heads, kv, cache, window):
    # the rows of a prompt and the same rows as sequences of one new token each, on the same pages; both are known within the tolerances
    # of kv_oracle.py, here from bounds on q, k and v instead of the sums themselves
    n = 4500
    pool = Pool(np.random.default_rng(dim), n // 64 + 2, kv, 64, dim, cache)
    table = pool.fill([n])
    kc, q = pool.upload(dev), queries(np.random.default_rng(3), n, heads, dim)
    a, b = Out(dev, q.shape, "f16"), Out(dev, q.shape, "f16")
    T.attention_prompt(dev, kc, sequences(dev, table, [n], [n]), At(dev, q), n, heads, a, window=window)
    T.attention_decode(dev, kc, sequences(dev, np.repeat(table, n, axis=0), np.arange(1, n + 1)), At(dev, q), heads, b, window=window)
    x, y = a.get().astype(np.float64), b.get().astype(np.float64)
    k, v = (np.abs(pool.tokens(name, table[0], n)) for name in "kv")
    group = heads // kv
    scores = dim ** -0.5 * np.einsum("rhd,hd->rh", np.abs(q).astype(np.float64), np.repeat(k.max(1), group, axis=0))   # above every sum of magnitudes
    d = (dim * 2.0 ** -23 + 2.0 ** -22) * scores + 2.0 ** -21
    most = np.repeat(v.max(1), group, axis=0)[None]
    each = ((2 * d + (n + 16) * 2.0 ** -23)[:, :, None] + 2.0 ** -25) * most
    tol = (2 * each + (PROMPT_STEP + DECODE_STEP) * most) * (1 + 2.0 ** -11) + half_step_f16(x) + half_step_f16(y)
    assert np.isfinite(x).all() and np.isfinite(y).all() and (np.abs(x - y) <= tol).all()
    # the first rows see few tokens, where a bound is as good as the sums
    want, exact_tol, _ = attend_rows(pool, table, [70], [70], q[:70], dim ** -0.5, window, PROMPT_STEP)
    check(a.get()[:70], want, exact_tol)


def test_all_rows_in_the_last_of_many_sequences(dev):
    new = [0] * 4100 + [70] + [0] * 200
    lengths = [0] * 4100 + [90] + [7] * 200
    pool = Pool(np.random.default_rng(7), 300, 2, 16, 64)
    run_prompt(dev, pool, pool.fill(lengths), lengths, new, 4, first=3, spare=2)


@pytest.mark.parametrize("least", [-1, -(1 << 31)])
def test_lengths_below_zero(dev, least):
    pool = Pool(np.random.default_rng(8), 10, 2, 16, 64)
    table = pool.fill([40, 0, 0])
    lengths = [40, least, least]
    for window in (0, 1, 30, 0xFFFFFFFF):
        run_decode(dev, pool, table, lengths, 4, window=window)
        run_prompt(dev, pool, table, lengths, [20, 0, 3], 4, window=window)


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dim,cache", [(64, "f16"), (128, "f16"), (256, "f16"), (128, "e4m3"), (256, "e4m3")])
def test_one_infinity_in_any_column_does_not_reach_the_rows_before_it(dev, dim, cache, wide):
    n = 40
    pool = Pool(np.random.default_rng(11), 4, 1, 16, dim, cache, scales=False)
    table, q = pool.fill([n], width=40 if wide else None), queries(np.random.default_rng(12), n, 1, dim)
    clean = run_prompt(dev, pool, table, [n], [n], 1, q=q)
    want, tol, _ = attend_rows(pool, table, [n], [n], q, dim ** -0.5, 0, PROMPT_STEP)
    bad = (0x7F, np.uint8) if cache == "e4m3" else (0x7C00, np.uint16)   # (e4m3 has no infinity: NaN)
    for column in range(dim):
        token = 1 + column % (n - 1)
        at = table[0, token // 16], 0, token % 16, column
        kept = pool.bits["v"][at]
        pool.bits["v"][at] = bad[0]
        out = Out(dev, q.shape, "f16")
        T.attention_prompt(dev, pool.upload(dev), sequences(dev, table, [n], [n]), At(dev, q), n, 1, out)
        pool.bits["v"][at] = kept
        got, others = out.get(), np.arange(dim) != column
        assert not np.isfinite(got[token:, 0, column]).any()
        check(got[:token], want[:token], tol[:token])
        check(got[token:][:, :, others], want[token:][:, :, others], tol[token:][:, :, others])
    assert np.array_equal(run_prompt(dev, pool, table, [n], [n], 1, q=q).view(np.uint16), clean.view(np.uint16))


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_rows_of_nothing_but_infinitely_low_scores_are_zeros(dev, dim, wide):
    n = 70
    pool = Pool(np.random.default_rng(13), 6, 1, 16, dim)
    table = pool.fill([n], width=40 if wide else None)
    q = np.abs(queries(np.random.default_rng(14), n, 2, dim)) + np.float16(0.25)
    pool.bits["k"][:, :, :, 3] = np.float16(-np.inf).view(np.uint16)
    kc, out, one = pool.upload(dev), Out(dev, q.shape, "f16"), Out(dev, (1, 2, dim), "f16")
    T.attention_prompt(dev, kc, sequences(dev, table, [n], [n]), At(dev, q), n, 2, out)
    T.attention_decode(dev, kc, sequences(dev, table, [n]), At(dev, q[:1]), 2, one)
    assert (out.get() == 0).all() and (one.get() == 0).all()


class Large:
    """A device array that no host array stands behind, cleared page by page."""

    def __init__(self, dev, elements, dtype):
        self.whole = T.GpuTensor(dev, (elements,), dtype)
        self.dtype, self.numel, self.ptr = dtype, elements, self.whole.ptr

    def part(self, dev, first, count):
        size = 1 if self.dtype == "u8" else 2
        out = np.empty(count, np.uint8 if self.dtype == "u8" else np.uint16)
        assert dev._l.twm_memcpy_d2h(dev.handle, out.ctypes.data, self.ptr + first * size, out.nbytes) == 0
        return out


@pytest.mark.parametrize("cache", ["f16", "e4m3"])
def test_pools_beyond_32_bit_offsets(dev, cache):
    # 5.2e9 elements each: the same rows stored on the pool's last pages and on the only ones of a small pool give the same bits
    kv, page, dim, heads, pages = 8, 256, 128, 16, 20000
    chunk, kind = kv * page * dim, "f16" if cache == "f16" else "u8"
    far_k, far_v = Large(dev, pages * chunk, kind), Large(dev, pages * chunk, kind)
    assert far_k.numel > 1 << 32
    near = Pool(np.random.default_rng(4), 4, kv, page, dim, cache, scales=False).upload(dev)
    far = T.KvCache(far_k, far_v, page, kv, dim)
    lengths, new = [300, 40], [300, 40]
    rows = (1.5 * np.random.default_rng(5).standard_normal((340, (heads + 2 * kv) * dim))).astype(np.float32)
    results = []
    for kc, table in ((near, [[2, 0], [1, -1]]), (far, [[pages - 1, 16383], [pages - 2, -1]])):
        seqs = sequences(dev, np.array(table, np.int32), lengths, new)
        q, out, one = Out(dev, (340, heads, dim), "f16"), Out(dev, (340, heads, dim), "f16"), Out(dev, (2, heads, dim), "f16")
        T.kv_append(dev, kc, seqs, At(dev, rows), 340, heads, q)
        T.attention_prompt(dev, kc, seqs, At(dev, q.get()), 340, heads, out)
        T.attention_decode(dev, kc, seqs, At(dev, q.get()[[299, 339]]), heads, one)
        results.append((out.get().view(np.uint16), one.get().view(np.uint16)))
    assert np.array_equal(results[0][0], results[1][0]) and np.array_equal(results[0][1], results[1][1])
    # and copied from one end of the pool to the other
    T.kv_copy_pages(dev, T.kv_layers([far]), [pages - 1, 16383], [1, pages - 3])
    dev.synchronize()
    for array in (far_k, far_v):
        assert np.array_equal(array.part(dev, chunk, chunk), array.part(dev, (pages - 1) * chunk, chunk))
        valid = 44 * dim   # (the second page holds 44 tokens of the first head)
        assert np.array_equal(array.part(dev, (pages - 3) * chunk, valid), array.part(dev, 16383 * chunk, valid))


def test_two_contexts_at_once(dev):
    # each has its own stream and scratch; shares, joins and single workgroups in turn
    rng = np.random.default_rng(6)
    with T.WarpDevice(0) as other:
        work = []
        for d, lengths in ((dev, [9000, 40, 700]), (other, [37, 8000, 5])):
            pool = Pool(rng, sum(-(-n // 64) for n in lengths), 2, 64, 64)
            table = pool.fill(lengths)
            q = queries(rng, 3, 6, 64)
            out, packed = Out(d, q.shape, "f16"), Out(d, q.shape, "f16")
            work.append((d, pool, table, lengths, q, pool.upload(d), sequences(d, table, lengths, [1, 1, 1]), At(d, q), out, packed))
        for _ in range(20):
            for d, _pool, _table, _lengths, _q, kc, seqs, q_dev, out, packed in work:
                T.attention_decode(d, kc, seqs, q_dev, 6, out)
                T.attention_prompt(d, kc, seqs, q_dev, 3, 6, packed)
        for d, pool, table, lengths, q, _kc, _seqs, _q_dev, out, packed in work:
            d.synchronize()
            for result, step in ((out, DECODE_STEP), (packed, PROMPT_STEP)):
                want, tol, _ = attend_rows(pool, table, lengths, [1, 1, 1], q, 0.125, 0, step)
                check(result.get(), want, tol)
