"""What perf/operators.py's calls return is in the order of torch's stream: read at once, without a synchronization, it is whole."""
import importlib.util
import os

import pytest
import torch

from tensorwarp_amd import build

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def operators():
    path = os.path.join(os.path.dirname(build.HERE), "perf", "operators.py")
    spec = importlib.util.spec_from_file_location("operators_under_test", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    module.own = True
    yield module
    if module._device is not None:
        module._device.close()


@pytest.mark.parametrize("name,out", [("gemm_4096x22016_m2048", "c"), ("norm_2048x4096", "normed"), ("sample_32x152064", "tokens")])
def test_results_read_at_once_are_whole(operators, name, out):
    # (the buffer is cleared by torch before each call and after each copy: a call that did not wait for the one, or a copy that did not
    # wait for the call, holds zeros)
    state = operators.prepare({c["name"]: c for c in operators.listed()}[name], 3)
    operators.run(state)
    torch.cuda.synchronize()
    want = state[out].clone()
    torch.cuda.synchronize()
    for _ in range(5):
        state[out].zero_()
        operators.run(state)
        got = state[out].clone()
        state[out].zero_()
        assert torch.equal(got, want)
