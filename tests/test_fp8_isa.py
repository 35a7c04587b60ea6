"""What the compiler made of the 8-bit path's and the sampler's kernels, checked on the CPU from the gfx950 assembly as
test_isa_health.py does for the older ones: registers, and the order of loads, waits and barriers that their sources pin."""
import re
import tempfile
from concurrent.futures import ThreadPoolExecutor

import pytest

from test_isa_health import assembly_of

FILES = ["twm_fp8_gemm.hip", "twm_fp8_rows.hip", "twm_sample.hip"]
# two workgroups of it share a compute unit, which leaves a wave 64 registers
SPILLS = {"8k_sampleILi8E": 20}   # bytes a lane


@pytest.fixture(scope="module")
def kernels():
    with tempfile.TemporaryDirectory() as d:
        with ThreadPoolExecutor(max_workers=len(FILES)) as pool:
            texts = list(pool.map(lambda f: assembly_of(f, d), FILES))
    found = {}
    for text in texts:
        for m in re.finditer(r"\n(_ZN3twm\w+):[^\n]*\n(.*?)s_endpgm", text, re.S):
            spill = re.search(r"\.set " + re.escape(m.group(1)) + r"\.private_seg_size, (\d+)", text)
            found[m.group(1)] = (m.group(2), int(spill.group(1)))
    return found


def test_no_kernel_spills(kernels):
    for kernel, forms in (("k_fp8_tileI", 5), ("k_fp8_rows_fewI", 16), ("k_fp8_splitsE", 1), ("k_fp8_rowsI", 12), ("k_fp8_normI", 12), ("k_sampleI", 2),
                          ("k_sample_largestE", 1), ("k_sample_limitsE", 1), ("k_sample_tokenE", 1)):
        assert sum("%d%s" % (len(kernel) - 1, kernel) in name for name in kernels) == forms, kernel
    for name, (_, scratch) in kernels.items():
        most = [b for part, b in SPILLS.items() if part in name]
        assert scratch <= (most[0] if most else 0), (name, scratch)


def test_tiles_change_hands_behind_whole_waits(kernels):
    # the start, the two copies of a step and the store: every load and every read of LDS has arrived before a buffer is given on
    tiles = [(name, body) for name, (body, _) in kernels.items() if "10k_fp8_tileI" in name]
    assert len(tiles) == 5
    for name, body in tiles:
        lines = [line.strip() for line in body.split("\n") if line.strip() and not line.strip().startswith((";", "."))]
        barriers = [i for i, line in enumerate(lines) if line == "s_barrier"]
        assert len(barriers) == 4, name
        for i in barriers:
            wait = max(j for j in range(i) if lines[j] == "s_waitcnt vmcnt(0) expcnt(0) lgkmcnt(0)")
            between = [line for line in lines[wait:i] if re.match(r"(ds|buffer|global|flat|s_load|s_cbranch|s_branch)_?", line)]
            assert not between, (name, between)   # (register work may come between the two)
        # nor is any product of a step missing
        s, tn, tm = (int(x) for x in re.search(r"10k_fp8_tileILi(\d+)ELi(\d+)ELi(\d+)E", name).groups())
        assert body.count("v_mfma") == 2 * tn * tm * (1 if s == 16 else 8), name


def test_eight_waves_issue_their_loads_one_by_one(kernels):
    # with every second product, not together (which held every wave of the unit up): between two of a step's operand loads there is a
    # matrix product, but where the next step's scales come in between
    (body,) = [body for name, (body, _) in kernels.items() if "10k_fp8_tileILi16ELi8ELi4ELi2ELi4E" in name]
    steps = re.split(r"\ts_barrier", body)[1:4]
    order = re.findall(r"v_mfma|buffer_load_dwordx4", "".join(steps))
    together = sum(a == b == "buffer_load_dwordx4" for a, b in zip(order, order[1:]))
    assert order.count("buffer_load_dwordx4") >= 16 and together <= 1


def test_few_rows_have_a_round_of_loads_in_flight(kernels):
    # up to 16 rows a wave's codes of W and A, for one or two blocks, are under way before any of them is waited for
    forms = [(name, body) for name, (body, _) in kernels.items() if re.search(r"14k_fp8_rows_fewILi1E\w+Lb0EEE", name)]
    assert len(forms) == 5
    for name, body in forms:
        nt, u = (int(x) for x in re.search(r"ILi1ELi(\d)ELi(\d)E", name).groups())
        first = re.search(r"global_load_dwordx4(?:(?!s_waitcnt vmcnt).)*", body, re.S).group(0)
        assert first.count("global_load_dwordx4") >= 2 * (nt + 1), (name, u)
