"""Captured steps of the paged key-value cache and its attention that share a context, and with it the scratch in which long sequences' parts meet: every
replay works on rows that the host has changed, into buffers that it has filled with something else, and what each graph leaves is compared, the first one's
too."""
import numpy as np
import pytest

import tensorwarp_amd as T
from kv_oracle import DECODE_STEP, PROMPT_STEP, Pool, attend_rows, check
from test_gpu_attention import ints, sequences
from test_gpu_fp8 import Out
from test_gpu_kv_cache import angles

pytestmark = pytest.mark.gpu

HEADS, KV, DIM, PAGE = 6, 2, 128, 16


@pytest.fixture(scope="module")
def dev():
    with T.WarpDevice(0) as d:
        yield d


class Step:
    """New tokens of two sequences, appended and attended to."""

    def __init__(self, dev, kc, cos_sin, table, lengths, new, prompt):
        self.dev, self.kc, self.cos_sin, self.table, self.lengths, self.new, self.prompt = dev, kc, cos_sin, table, lengths, new, prompt
        self.n = sum(new)
        self.q, self.out = Out(dev, (self.n, HEADS, DIM), "f16"), Out(dev, (self.n, HEADS, DIM), "f16")
        self.qkv = T.GpuTensor.zeros(dev, (self.n, (HEADS + 2 * KV) * DIM), "f32")
        self.seqs = sequences(dev, table, lengths, new)

    def launch(self):
        T.kv_append(self.dev, self.kc, self.seqs, self.qkv, self.n, HEADS, self.q, cos_sin=self.cos_sin, positions=6000, rotary_dim=DIM)
        if self.prompt:
            T.attention_prompt(self.dev, self.kc, self.seqs, self.q, self.n, HEADS, self.out)
        else:
            T.attention_decode(self.dev, self.kc, self.seqs, self.q, HEADS, self.out)

    def renew(self, rng):
        self.qkv.copy_from_host((1.5 * rng.standard_normal((self.n, (HEADS + 2 * KV) * DIM))).astype(np.float32))
        for buffer in (self.q, self.out):
            buffer.whole.copy_from_host(buffer.fill)

    def expect(self, pool):
        want, tol, _ = attend_rows(pool, self.table, self.lengths, self.new, self.q.get(), DIM ** -0.5, 0, PROMPT_STEP if self.prompt else DECODE_STEP)
        check(self.out.get(), want, tol)


@pytest.mark.parametrize("cache", ["f16", "e4m3"])
@pytest.mark.parametrize("first,second", [("decode", "prompt"), ("prompt", "decode"), ("decode", "decode"), ("prompt", "prompt")])
def test_both_of_two_captured_steps_leave_their_results(dev, first, second, cache):
    # (a step's tokens lie behind those that the one before sees, so that both are still known after the last replay)
    rng = np.random.default_rng(41)
    pool = Pool(rng, 800, KV, PAGE, DIM, cache)
    table = pool.fill([5000, 3000], 320)
    for row in range(2):
        for i in np.flatnonzero(table[row] < 0):
            table[row, i] = pool.free.pop()
    kc, cos_sin = pool.upload(dev), T.GpuTensor.from_host(dev, angles(6000, DIM))
    steps, lengths = [], [5000, 3000]
    for kind in (first, second):
        new = [1, 1] if kind == "decode" else [2, 3]
        lengths = [a + b for a, b in zip(lengths, new)]
        steps.append(Step(dev, kc, cos_sin, table, lengths, new, kind == "prompt"))
    for step in steps:
        step.renew(rng)
        step.launch()   # (once before, as a serving program does)
    dev.synchronize()
    graphs = [T.GraphCapture.record_with_device(dev, step.launch) for step in steps]
    other = Step(dev, kc, cos_sin, table, [4000, 2000], [1, 1], False)
    for order in ((0, 1), (1, 0), (0, 1, 0, 1), (1, 0, 0)):
        for step in steps:
            step.renew(rng)
        for i in order:
            graphs[i].replay()
        if order[0] == 1:   # (the second step saw the first one's tokens as they were before)
            graphs[1].replay()
        dev.synchronize()
        pool.download()
        for step in steps:
            step.expect(pool)
        other.renew(rng)   # the program's own work in between: tokens that both see
        other.launch()
        dev.synchronize()
        pool.download()
        other.expect(pool)
