"""Rows into the paged key-value cache, pages to other pages, and the calls of the cache together, through the C ABI against numpy in
64 bits."""
import numpy as np
import pytest

import tensorwarp_amd as T
from kv_oracle import DECODE_STEP, E4M3, PROMPT_STEP, Pool, attend_rows, check, half_step_f16
from test_gpu_attention import ints, sequences
from test_gpu_fp8 import At, Out

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    with T.WarpDevice(0) as d:
        yield d


def rotated(x, position, table, rotary, interleaved):
    """x [heads, dim] in 64 bits, and how far f32 may be off: two products and a sum, of which a fused step rounds one."""
    y, err, half = x.copy(), np.zeros_like(x), rotary // 2
    if rotary == 0:
        return y, err
    if position >= len(table):
        y[:] = np.where(np.arange(x.shape[1]) < rotary, np.nan, y)
        return y, err
    c, s = table[position, :half].astype(np.float64), table[position, half:].astype(np.float64)
    a, b = (slice(0, rotary, 2), slice(1, rotary, 2)) if interleaved else (slice(0, half), slice(half, rotary))
    y[:, a], y[:, b] = x[:, a] * c - x[:, b] * s, x[:, b] * c + x[:, a] * s
    err[:, a], err[:, b] = (np.abs(x[:, a] * c) + np.abs(x[:, b] * s)) * 2.0 ** -23, (np.abs(x[:, b] * c) + np.abs(x[:, a] * s)) * 2.0 ** -23
    return y, err


def angles(positions, rotary):
    at = np.arange(positions)[:, None] * 10000.0 ** (-np.arange(rotary // 2) / max(1, rotary // 2))
    return np.concatenate([np.cos(at), np.sin(at)], axis=1).astype(np.float32)


def check_cached(pool, name, page, token, y, err):
    """The heads' values y [kv_heads, dim], known within err, at one token's place."""
    got = pool.bits[name][page, :, token]
    if pool.cache == "f16":
        v = got.view(np.float16).astype(np.float64)
        nan = np.isnan(y)
        assert np.array_equal(np.isnan(v), nan)
        with np.errstate(invalid="ignore"):
            over = np.abs(y) >= 65520
        assert np.array_equal(np.isinf(v), over)
        ok = ~nan & ~over
        assert (np.abs(v - y) <= half_step_f16(y) + err * (1 + 2.0 ** -10))[ok].all()
        return
    scale = np.ones(len(y)) if pool.scales[name] is None else pool.scales[name].astype(np.float64)
    u, off = y / scale[:, None], err / scale[:, None] + 2.0 ** -23 * np.abs(y / scale[:, None])
    nan = np.isnan(u)
    assert np.array_equal(got & 0x7F == 0x7F, nan)
    u = np.clip(u, -448, 448)
    assert (np.abs(E4M3[got] - u) <= np.maximum(2.0 ** -4 * np.abs(u), 2.0 ** -10) + off)[~nan].all()


def run_append(dev, pool, table, lengths, new, heads, x="f16", rotary=None, interleaved=False, positions=None, more=0, skip=0, starts=True, spare=0):
    rng, (pages, kv, page, dim) = np.random.default_rng(7), pool.shape
    rotary = dim if rotary is None else rotary
    rows, width = sum(new), (heads + 2 * kv) * dim
    cos_sin = angles(max([1] + list(lengths)) if positions is None else positions, rotary)
    qkv = (2 * rng.standard_normal((rows + spare, width + more))).astype(np.float16 if x == "f16" else np.float32)
    before = {name: pool.bits[name].copy() for name in "kv"}
    out = Out(dev, (rows + spare, heads, dim), "f16")
    cache = pool.upload(dev)
    T.kv_append(dev, cache, sequences(dev, table, lengths, new if starts else None), At(dev, qkv, skip), rows + spare, heads, out,
                cos_sin=At(dev, cos_sin, skip) if rotary else None, positions=len(cos_sin), rotary_dim=rotary, interleaved=interleaved,
                qkv_stride=width + more if more else 0)
    pool.download()
    q, row, written = out.get(), 0, np.zeros((pages, page), bool)
    for s, (n, length) in enumerate(zip(new, lengths)):
        for i in range(n):
            position = length - n + i
            if position < 0:
                assert (q[row].view(np.uint16) == 12345).all()
                row += 1
                continue
            y = qkv[row, :width].astype(np.float64).reshape(-1, dim)
            turned, err = rotated(y[:heads + kv], position, cos_sin, rotary, interleaved)
            want = turned[:heads]
            assert np.array_equal(np.isnan(q[row]), np.isnan(want))
            ok = ~np.isnan(want)
            assert (np.abs(q[row].astype(np.float64) - want) <= half_step_f16(want) + err[:heads] * (1 + 2.0 ** -10))[ok].all()
            if position // page < table.shape[1] and 0 <= table[s, position // page] < pages:
                p = table[s, position // page]
                check_cached(pool, "k", p, position % page, turned[heads:], err[heads:])
                check_cached(pool, "v", p, position % page, y[heads + kv:], np.zeros((kv, dim)))
                written[p, position % page] = True
            row += 1
    assert (q[row:].view(np.uint16) == 12345).all()
    for name in "kv":   # every other place is as it was
        same = (pool.bits[name] == before[name]).all(axis=(1, 3))
        assert same[~written].all()


APPENDS = [([1], [1]), ([1], [500]), ([37], [37]), ([20, 0, 1, 64], [20, 3, 130, 100]), ([1, 1, 1], [16, 17, 1]), ([130], [300])]


@pytest.mark.parametrize("x", ["f16", "f32"])
@pytest.mark.parametrize("cache", ["f16", "e4m3"])
@pytest.mark.parametrize("dim,page,heads,kv", [(64, 16, 14, 2), (128, 64, 28, 4), (256, 32, 2, 1), (128, 256, 9, 3)])
@pytest.mark.parametrize("new,lengths", APPENDS)
def test_append(dev, new, lengths, dim, page, heads, kv, cache, x):
    pool = Pool(np.random.default_rng(dim + sum(new)), 60 if page < 64 else 12, kv, page, dim, cache)
    run_append(dev, pool, pool.fill(lengths), lengths, new, heads, x)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rotary", [0, 16, 48, 64, 128])
@pytest.mark.parametrize("cache", ["f16", "e4m3"])
def test_rotations(dev, cache, rotary, interleaved):
    pool = Pool(np.random.default_rng(rotary), 40, 2, 16, 128, cache, scales=rotary != 48)
    run_append(dev, pool, pool.fill([70, 33]), [70, 33], [70, 5], 6, "f32", rotary, interleaved)


def test_far_positions_and_positions_beyond_the_table(dev):
    pool = Pool(np.random.default_rng(1), 1300, 1, 16, 64)
    run_append(dev, pool, pool.fill([20000]), [20000], [9], 2, "f32")
    pool = Pool(np.random.default_rng(2), 40, 2, 16, 64)
    run_append(dev, pool, pool.fill([100, 30]), [100, 30], [60, 30], 4, "f16", positions=70)
    run_append(dev, pool, pool.fill([100]), [100], [60], 4, "f16", rotary=32, positions=0)


@pytest.mark.parametrize("more,skip,x", [(3, 1, "f16"), (0, 3, "f32"), (8, 5, "f16")])
def test_rows_of_any_stride_at_any_address(dev, more, skip, x):
    pool = Pool(np.random.default_rng(3), 40, 2, 16, 64)
    run_append(dev, pool, pool.fill([50, 9]), [50, 9], [50, 1], 6, x, more=more, skip=skip)


def test_rows_that_are_not_stored(dev):
    # more rows than tokens, pages outside the pool, positions behind the table, rows behind the last sequence
    pool = Pool(np.random.default_rng(4), 40, 2, 16, 64)
    lengths = [20, 3, -4, 100]
    table = pool.fill([20, 3, 0, 60])
    table[0, 1] = 40
    table[3, 0] = -9
    run_append(dev, pool, table, lengths, [20, 7, 2, 100], 4, spare=3)


def test_one_row_a_sequence(dev):
    lengths = [5, 1, 64, 0, 200]
    pool = Pool(np.random.default_rng(5), 40, 2, 16, 128, "e4m3")
    run_append(dev, pool, pool.fill(lengths), lengths, [1] * 5, 4, starts=False)


def test_many_sequences(dev):
    # more than a workgroup has threads, empty ones among them
    rng = np.random.default_rng(6)
    new = list(rng.integers(0, 3, 700))
    lengths = [n + int(rng.integers(0, 20)) for n in new]
    pool = Pool(rng, sum(-(-n // 16) for n in lengths) + 1, 1, 16, 64)
    run_append(dev, pool, pool.fill(lengths), lengths, new, 1, "f32")


def test_thousands_of_sequences(dev):
    # more than the square of a workgroup's threads would hold in one look, and rows of one among empty ones
    rng = np.random.default_rng(9)
    new = list(rng.integers(0, 2, 5000))
    lengths = [n + int(rng.integers(0, 3)) for n in new]
    pool = Pool(rng, sum(-(-n // 16) for n in lengths) + 1, 1, 16, 64)
    run_append(dev, pool, pool.fill(lengths), lengths, new, 1, "f32")
    new, lengths = [0] * 4500 + [30] + [0] * 77, [0] * 4500 + [50] + [2] * 77
    run_append(dev, pool := Pool(rng, 90, 1, 16, 64), pool.fill(lengths), lengths, new, 1)


@pytest.mark.parametrize("least", [-1, -(1 << 31)])
def test_rows_of_lengths_below_zero_are_not_stored(dev, least):
    pool = Pool(np.random.default_rng(10), 8, 2, 16, 64)
    run_append(dev, pool, pool.fill([20, 0, 0]), [20, least, least], [5, 2, 1], 4)


def test_values_beyond_f16_and_e4m3(dev):
    for cache in ("f16", "e4m3"):
        pool = Pool(np.random.default_rng(8), 4, 1, 16, 64, cache, scales=False)
        table, lengths = pool.fill([4]), [4]
        qkv = np.zeros((4, 3 * 64), np.float32)
        qkv[0, 64:68] = [1e6, -1e6, np.inf, -np.inf]
        qkv[1, 128:132] = [65519.0, 65520.0, np.nan, 449.0]
        qkv[2, :4] = [1e9, -1e9, np.nan, 1e-9]
        out = Out(dev, (4, 64), "f16")
        T.kv_append(dev, pool.upload(dev), sequences(dev, table, lengths, [4]), At(dev, qkv), 4, 1, out)
        pool.download()
        k, v, q = pool.bits["k"][table[0, 0], 0, 0, :4], pool.bits["v"][table[0, 0], 0, 1, :4], out.get()[2, :4]
        if cache == "f16":
            assert np.array_equal(k.view(np.float16), np.array([np.inf, -np.inf, np.inf, -np.inf], np.float16))
            assert np.array_equal(v.view(np.float16), np.array([65504, np.inf, np.nan, 449], np.float16), equal_nan=True)
        else:
            assert np.array_equal(E4M3[k], [448, -448, 448, -448])
            assert np.array_equal(E4M3[v], [448, 448, np.nan, 448], equal_nan=True)
        assert np.isposinf(q[0]) and np.isneginf(q[1]) and np.isnan(q[2]) and q[3] == 0


# ---- pages -------------------------------------------------------------------------------------------------------------


def run_copy(dev, layers, pairs, pages, kv, page, dim, cache):
    rng = np.random.default_rng(pairs)
    pools, caches = [], []
    for _ in range(layers):
        p = Pool(rng, pages, kv, page, dim, cache)
        for name in "kv":
            p.bits[name] = rng.integers(0, 256, p.bits[name].nbytes, dtype=np.uint8).view(p.bits[name].dtype).reshape(p.shape)
        pools.append(p)
        caches.append(p.upload(dev))
    order = rng.permutation(pages)
    targets, sources = order[:pairs], rng.choice(order[pairs:], pairs)   # (a source may be named more than once)
    T.kv_copy_pages(dev, T.kv_layers(caches), sources, targets)
    for p in pools:
        before = {name: p.bits[name].copy() for name in "kv"}
        p.download()
        for name in "kv":
            before[name][targets] = before[name][sources]
            assert np.array_equal(p.bits[name], before[name])


@pytest.mark.parametrize("layers,pairs,pages,kv,page,dim,cache", [
    (1, 1, 3, 1, 16, 64, "e4m3"), (1, 1, 2, 1, 16, 64, "f16"), (28, 1, 5, 4, 16, 128, "f16"), (3, 20, 41, 3, 16, 64, "e4m3"), (2, 5, 11, 5, 256, 64, "f16"),
    (70, 3, 8, 1, 16, 64, "f16"), (1, 700, 1500, 1, 16, 64, "e4m3"), (2, 330, 700, 1, 32, 64, "f16")])
def test_copies(dev, layers, pairs, pages, kv, page, dim, cache):
    run_copy(dev, layers, pairs, pages, kv, page, dim, cache)


def test_a_captured_copy_copies_what_is_there_at_its_replay(dev):
    rng = np.random.default_rng(12)
    pools = [Pool(rng, 9, 2, 16, 64) for _ in range(3)]
    layers = T.kv_layers([p.upload(dev) for p in pools])
    sources, targets = [4, 4, 0], np.array([1, 8, 3])
    T.kv_copy_pages(dev, layers, sources, targets)   # (once before)
    graph = T.GraphCapture.record_with_device(dev, lambda: T.kv_copy_pages(dev, layers, sources, targets))
    for _ in range(4):
        for p in pools:
            for name in "kv":
                p.bits[name] = rng.integers(0, 1 << 16, p.shape).astype(np.uint16)
                p.dev[name].copy_from_host(p.bits[name])
        graph.replay()
        dev.synchronize()
        for p in pools:
            before = {name: p.bits[name].copy() for name in "kv"}
            p.download()
            for name in "kv":
                before[name][targets] = before[name][sources]
                assert np.array_equal(p.bits[name], before[name])
        T.kv_copy_pages(dev, layers, [2], [5])   # eager work in between


# ---- together ----------------------------------------------------------------------------------------------------------


class Server:
    """A layer's attention as a serving program runs it, on the device, and the same on the host."""

    def __init__(self, dev, cache, heads=6, kv=2, dim=128, page=16, pages=60):
        self.dev, self.heads, self.kv, self.dim = dev, heads, kv, dim
        self.rng = np.random.default_rng(31)
        self.pool = Pool(self.rng, pages, kv, page, dim, cache)
        self.cache = self.pool.upload(dev)
        self.cos_sin = T.GpuTensor.from_host(dev, angles(400, dim))

    def rows(self, n):
        return (1.5 * self.rng.standard_normal((n, (self.heads + 2 * self.kv) * self.dim))).astype(np.float32)

    def buffers(self, n):
        return Out(self.dev, (n, self.heads, self.dim), "f16"), Out(self.dev, (n, self.heads, self.dim), "f16")

    def launch(self, seqs, qkv, n, q, out, prompt, window=0):
        T.kv_append(self.dev, self.cache, seqs, qkv, n, self.heads, q, cos_sin=self.cos_sin, positions=400, rotary_dim=self.dim)
        if prompt:
            T.attention_prompt(self.dev, self.cache, seqs, q, n, self.heads, out, window=window)
        else:
            T.attention_decode(self.dev, self.cache, seqs, q, self.heads, out, window=window)

    def expect(self, q, out, table, lengths, new, prompt, window=0):
        # from what the cache holds now (its contents are checked by themselves above)
        self.pool.download()
        want, tol, _ = attend_rows(self.pool, table, lengths, new, q.get(), self.dim ** -0.5, window, PROMPT_STEP if prompt else DECODE_STEP)
        check(out.get(), want, tol)
        return want

    def step(self, table, lengths, new, prompt, window=0):
        n = sum(new)
        q, out = self.buffers(n)
        self.launch(sequences(self.dev, table, lengths, new), T.GpuTensor.from_host(self.dev, self.rows(n)), n, q, out, prompt, window)
        return self.expect(q, out, table, lengths, new, prompt, window)


@pytest.mark.parametrize("cache", ["f16", "e4m3"])
def test_prompts_forks_and_single_tokens(dev, cache):
    # two prompts; a third in two pieces; the first is forked with its last page copied; then all of them, token by token
    s = Server(dev, cache)
    table = np.full((4, 8), -1, np.int32)
    pages = iter(range(60))
    for row, count in ((0, 3), (1, 1), (2, 7)):
        table[row, :count] = [next(pages) for _ in range(count)]
    s.step(table[:2], [45, 12], [45, 12], True)
    s.step(table[2:3], [70], [70], True)
    s.step(table[2:3], [101], [31], True)
    table[3, :2] = table[0, :2]
    table[3, 2] = next(pages)
    T.kv_copy_pages(dev, T.kv_layers([s.cache]), [int(table[0, 2])], [int(table[3, 2])])
    lengths = [45, 12, 101, 45]
    for _ in range(6):
        for r in range(4):
            if lengths[r] % 16 == 0:
                table[r, lengths[r] // 16] = next(pages)
            lengths[r] += 1
        s.step(table, lengths, [1] * 4, False)
    # drafts: three tokens each at once, verified by the packed form
    for r in range(4):
        while table[r, (lengths[r] + 2) // 16] < 0:
            table[r, (lengths[r] + 2) // 16] = next(pages)
        lengths[r] += 3
    s.step(table, lengths, [3] * 4, True)


@pytest.mark.parametrize("cache", ["f16", "e4m3"])
def test_a_captured_step_reads_lengths_and_tables_at_its_replay(dev, cache):
    s = Server(dev, cache)
    table = np.arange(60, dtype=np.int32)[:60].reshape(3, 20)
    lengths = np.array([1, 40, 200], np.int32)
    lengths_dev, table_dev, qkv = ints(dev, lengths), ints(dev, table), T.GpuTensor.from_host(dev, s.rows(3))
    s.step(table, [0, 39, 199], [0, 39, 199], True)
    seqs = T.KvSequences(table_dev, lengths_dev, 3, 20)
    q, out = s.buffers(3)
    s.launch(seqs, qkv, 3, q, out, False)   # (once before, as a serving program does)
    graph = T.GraphCapture.record_with_device(dev, lambda: s.launch(seqs, qkv, 3, q, out, False))
    for _ in range(4):
        qkv.copy_from_host(s.rows(3))
        lengths_dev.copy_from_host(lengths)
        graph.replay()
        dev.synchronize()
        s.expect(q, out, table, list(lengths), [1, 1, 1], False)
        s.step(table, [30, 40, 200], [1, 1, 1], False)   # eager work in between
        lengths += np.array([25, 1, 17], np.int32)


def test_two_captured_steps_take_turns(dev):
    # two graphs of one context share its scratch, one after the other
    s = Server(dev, "f16", pages=400)
    table = np.arange(400, dtype=np.int32).reshape(2, 200)
    s.cos_sin = T.GpuTensor.from_host(dev, angles(400, s.dim))
    s.step(table[:, :25], [390, 300], [390, 300], True)
    graphs = []
    for new, lengths in (([1, 1], [391, 301]), ([2, 3], [393, 304])):
        n, prompt = sum(new), new[0] > 1
        q, out = s.buffers(n)
        qkv, seqs = T.GpuTensor.from_host(dev, s.rows(n)), sequences(dev, table, lengths, new)
        s.launch(seqs, qkv, n, q, out, prompt)
        graph = T.GraphCapture.record_with_device(dev, lambda: s.launch(seqs, qkv, n, q, out, prompt))
        graphs.append((graph, q, out, lengths, new, prompt, (qkv, seqs)))
    for _ in range(3):
        for graph, q, out, lengths, new, prompt, _keep in graphs:
            graph.replay()
        dev.synchronize()
        for graph, q, out, lengths, new, prompt, _keep in graphs[1:]:
            s.expect(q, out, table, lengths, new, prompt)


def test_on_a_stream_of_the_callers(dev):
    stream = dev._l.twm_stream_create(dev.handle)
    dev.with_stream(stream)
    try:
        s = Server(dev, "f16")
        table = np.arange(60, dtype=np.int32).reshape(3, 20)
        for name in "kv":   # (uploads are synchronous; downloads wait for the stream's work)
            assert s.pool.bits[name].size
        q, out = s.buffers(60)
        s.launch(sequences(dev, table, [20, 20, 20], [20, 20, 20]), T.GpuTensor.from_host(dev, s.rows(60)), 60, q, out, True)
        assert dev._l.twm_stream_sync(dev.handle, stream) == 0
        s.expect(q, out, table, [20, 20, 20], [20, 20, 20], True)
    finally:
        dev.synchronize()
        dev.with_stream(None)
        dev._l.twm_stream_destroy(dev.handle, stream)
