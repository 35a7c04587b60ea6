"""Attention over a paged key-value cache with infinite values on tokens that a row sees, however little these weigh: the column is that infinity, or NaN
where two of them differ, and the other columns are what they would be."""
import numpy as np
import pytest

import tensorwarp_amd as T
from kv_oracle import DECODE_STEP, PROMPT_STEP, Pool, half_step_f16
from test_gpu_attention import sequences
from test_gpu_attention_magnitudes import run

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    with T.WarpDevice(0) as d:
        yield d


def bits(x):
    return np.float16(x).view(np.uint16)


def built(n, dim, width, scores, infinite):
    """One sequence whose token t scores scores[t] with queries of ones in one place; infinite: {(token, column): value}."""
    pool = Pool(np.random.default_rng(n + dim), -(-n // 16) + 3, 2, 16, dim)
    table = pool.fill([n], width)
    for t in range(n):
        at = table[0, t // 16], slice(None), t % 16
        pool.bits["k"][at] = 0
        pool.bits["k"][at][:, 6] = bits(scores[t])
    v = pool.tokens("v", table[0], n)[0].copy()
    pool.bits["v"][:, 1] = pool.bits["v"][:, 0]   # (both key-value heads alike)
    for (t, column), value in infinite.items():
        pool.bits["v"][table[0, t // 16], :, t % 16, column] = bits(value)
    return pool, table, v


def expect(got, v, scores, infinite, first_row, step):
    """Rows of tokens first_row .. n - 1."""
    n, dim = v.shape
    columns = np.array([c for c in range(dim) if c not in {c for _, c in infinite}])
    top = np.maximum.accumulate(scores)
    for i, row in enumerate(range(first_row, n)):
        p = np.exp(scores[:row + 1] - top[row])
        total = p.sum()
        want, magnitude = p @ v[:row + 1] / total, p @ np.abs(v[:row + 1]) / total
        # scores are exact; a difference of up to 700 times the scale in base 2, off by 2^-22 of itself, where its weight is not yet nothing (2^7 of it)
        tol = (step + 2.0 ** -14 + (n + 16) * 2.0 ** -23) * magnitude + 2.0 ** -33 * np.abs(v[:row + 1]).sum(0)
        off = np.abs(got[i][:, columns] - want[columns]) / (tol + half_step_f16(want))[columns]
        assert off.max() <= 1.0, (row, off.max())
        for column in {c for _, c in infinite}:
            seen = {float(x) for (t, c), x in infinite.items() if c == column and t <= row}
            if not seen:
                assert np.isfinite(got[i][:, column]).all(), (row, column)
            elif len(seen) == 1:
                assert (got[i][:, column] == seen.pop()).all(), (row, column, got[i][:, column])
            else:
                assert np.isnan(got[i][:, column]).all(), (row, column)


def both(dev, pool, table, v, scores, infinite, n, new, heads=4):
    dim = v.shape[1]
    q = np.zeros((n, heads, dim), np.float16)
    q[:, :, 6] = 1.0
    kc = pool.upload(dev)
    expect(run(dev, kc, sequences(dev, table, [n], [new]), q[:new], heads, scale=1.0), v, scores, infinite, n - new, PROMPT_STEP)
    expect(run(dev, kc, sequences(dev, table, [n]), q[:1], heads, scale=1.0), v, scores, infinite, n - 1, DECODE_STEP)


INF = float("inf")


@pytest.mark.parametrize("width", [None, 400])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("behind", [10.0, 24.0, 40.0, 200.0])
@pytest.mark.parametrize("n,at,heavy", [(40, 20, 3), (40, 3, 20), (400, 10, 0), (400, 1, 130), (400, 200, 70), (400, 399, 5), (300, 5, 299), (330, 70, 69)])
def test_an_infinite_value_of_a_token_that_weighs_little(dev, n, at, heavy, behind, dim, width):
    # (before and behind the token that weighs most, in its tile and in others: the reference moves after it, or never does)
    scores = np.zeros(n)
    scores[heavy] = behind
    infinite = {(at, 5): INF, (at, 40): -INF}
    pool, table, v = built(n, dim, width, scores, infinite)
    both(dev, pool, table, v, scores, infinite, n, n)


@pytest.mark.parametrize("width", [None, 2000])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 7, 90])
@pytest.mark.parametrize("at,heavy", [(100, 3000), (3000, 100), (2990, 3040), (3, 5)])
def test_where_tokens_are_shared_out_and_joined(dev, at, heavy, new, dim, width):
    n = 3100
    scores = np.zeros(n)
    scores[heavy] = 300.0
    infinite = {(at, 5): INF, (at, 40): -INF, (at + 700 if at < 2000 else at - 700, 7): INF}
    pool, table, v = built(n, dim, width, scores, infinite)
    both(dev, pool, table, v, scores, infinite, n, new)


@pytest.mark.parametrize("width", [None, 400])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_scores_that_rise_behind_it_and_two_of_a_column(dev, dim, width):
    # every token outweighs those before it by e^3; column 5 is infinite from the third token on, 9 NaN once the other sign is seen, 11 has twice the same
    n = 220
    scores = 3.0 * np.arange(n)
    infinite = {(2, 5): INF, (70, 9): INF, (130, 9): -INF, (1, 11): -INF, (200, 11): -INF}
    pool, table, v = built(n, dim, width, scores, infinite)
    both(dev, pool, table, v, scores, infinite, n, n)


@pytest.mark.parametrize("width", [None, 400])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("size", [2000.0, 40000.0])
def test_beside_scores_of_millions(dev, size, dim, width):
    n = 200
    scores = np.zeros(n)
    scores[[30, 140]] = size
    infinite = {(10, 5): INF, (150, 6): -INF}
    pool, table, v = built(n, dim, width, scores, infinite)
    both(dev, pool, table, v, scores, infinite, n, n)


@pytest.mark.parametrize("width", [None, 2000])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("n,new", [(50, 50), (300, 300), (3100, 5)])
def test_rows_of_nothing_but_infinitely_low_scores_are_zeros_beside_any_value(dev, n, new, dim, width):
    pool, table, _ = built(n, dim, width, np.full(n, -np.inf), {(3, 5): INF, (n - 1, 6): float("nan"), (n // 2, 7): -INF})
    q = np.zeros((new, 4, dim), np.float16)
    q[:, :, 6] = 1.0
    kc = pool.upload(dev)
    assert (run(dev, kc, sequences(dev, table, [n], [new]), q, 4, scale=1.0) == 0).all()
    assert (run(dev, kc, sequences(dev, table, [n]), q[:1], 4, scale=1.0) == 0).all()
